// layernorm.cu -- layer norm whose weight and bias learn: forward with the 8-bit checkpoint of its
// input and the 8-bit form of its result, backward from either form of the input, with the sums
// over the rows that are the weight's and the bias's gradients.
//
// Both passes read every element once and are bound by HBM.  A row is held in registers, four
// columns a lane and NCH blocks of 128 columns a warp, by W warps; variance is the mean square of
// the differences from the mean, taken from those registers (no cancellation as in E[x^2] -
// E[x]^2, and no second read).  All statistics and sums are fp32.
#include <atomic>
#include <type_traits>

#include "ckpt8.cuh"

namespace act {

namespace {

using namespace c8;

// ---------------------------------------------------------------------------------------
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
template <typename T, int W, int NCH, int G, bool VEC>
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
        if (p.x8.q) {
            // a value that is not finite makes the sum of squares so: one test a row
            const bool bad = !(sq < __int_as_float(0x7f800000));
            uint32_t scale = 0;
#pragma unroll
            for (int k = 0; k < NCH; ++k) {
                float f[4];
                unpairs(v[k], f);
                const uint32_t s =
                    scale_bits(__reduce_max_sync(FULL_WARP, bad ? largest_finite(f) : largest(f)), p.x8.e4m3);
                store_codes<VEC>(x8 + k * W * BLOCK, left - k * W * BLOCK, encode4(f, inverse_pow2(s), p.x8.e4m3, bad));
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

// ---------------------------------------------------------------------------------------
// Backward.  A CTA's G row groups of W warps walk over rows; each lane keeps the sums dw and db of
// its own columns in registers over all rows of its group, the groups add theirs in order in
// shared memory, and each CTA leaves one row of partial sums that a second kernel adds in CTA
// order.  Every lane copies its own pieces of the next BWD_DEPTH rows into shared memory ahead of
// their use (cp.async: nobody else reads them, so no barrier is needed), which keeps enough
// bytes in flight at one CTA of 16 warps an SM, all that the sums' registers leave room for.
constexpr int BWD_WARPS = 16;
constexpr int BWD_NCH = 4;  // blocks of 128 columns a warp holds at most
constexpr int BWD_DEPTH = 4;

struct BwdParams {
    long rows, ldy, ldx, lddx;  // strides in bytes
    const char *dy, *x, *add;
    char* dx;
    int dy_half, x_half, dx_wide, dx_half, dim;
    const float *w, *mean, *rstd, *scale;
    long lds;
    float inv_dim;
    float* part;  // [CTAs][2][dim]
};

template <int BYTES>
__device__ __forceinline__ void copy_ahead(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}

// four elements of B bytes that a lane put into shared memory
template <int B>
__device__ __forceinline__ void read4(const unsigned char* p, bool half, float v[4]) {
    if (B == 4) unpack4(*reinterpret_cast<const float4*>(p), v, float());
    else if (half) unpack4(*reinterpret_cast<const uint2*>(p), v, f16());
    else unpack4(*reinterpret_cast<const uint2*>(p), v, __nv_bfloat16());
}

// DB, XB: bytes of an element of dy and of the kept input (1: codes, E4M3 or I8); AHEAD: lanes copy
// ahead, everything moves four elements at a time and w stays in registers.  Columns past the row's end read as x = 0 and dy = 0,
// so that they add nothing to any sum whatever their h is.
template <int DB, int XB, bool E4M3, int W, int NCH, bool AHEAD>
__global__ void __launch_bounds__(BWD_WARPS * 32) ln_bwd_kernel(const BwdParams p) {
    constexpr int G = BWD_WARPS / W, THREADS = BWD_WARPS * 32, NEXT = W * BLOCK;
    // a stage: per block a lane's four of dy and four of x
    constexpr int X_OFF = NCH * 4 * DB * THREADS, STAGE = X_OFF + NCH * 4 * XB * THREADS;
    constexpr int DEPTH = STAGE * BWD_DEPTH <= 160 * 1024 ? BWD_DEPTH : 2;
    __shared__ float2 slots[2][G][W];
    extern __shared__ __align__(16) unsigned char room[];  // the stages; at the end [2][dim] sums
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, grp = warp / W, wid = warp % W, t = threadIdx.x;
    const int first_c = wid * BLOCK + first_col<AHEAD>(lane), left = p.dim - first_c;
    uint64_t dw[NCH][2] = {}, db[NCH][2] = {};
    const long step = (long)gridDim.x * G, first = (long)blockIdx.x * G + grp;
    const char *dy = p.dy + first * p.ldy + first_c * DB, *x = p.x + first * p.ldx + first_c * XB;
    // lane k fetches block k's scale of the next row; every lane its mean and rstd
    const bool scales = XB == 1 && lane < NCH && (lane * W + wid) * BLOCK < p.dim;
    const float *scale_at = p.scale + (scales ? (long)(lane * W + wid) * p.lds : 0) + first, *mean_at = p.mean + first,
                *rstd_at = p.rstd + first;
    float next_scale = 0.f, next_mean = 0.f, next_rstd = 0.f;
    auto fetch = [&](bool any) {
        if (any) {
            if (scales) next_scale = *scale_at;
            next_mean = *mean_at;
            next_rstd = *rstd_at;
        }
        scale_at += step;
        mean_at += step;
        rstd_at += step;
    };
    uint64_t w2[AHEAD ? NCH : 1][2];
    if (AHEAD)
#pragma unroll
        for (int k = 0; k < NCH; ++k) {
            float f[4] = {1.f, 1.f, 1.f, 1.f};
            if (p.w) load4_const<true>(p.w + first_c + k * NEXT, left - k * NEXT, f);
            pairs(f, w2[k]);
        }
    const uint32_t ring = smem_u32(room) + t * 4 * DB, xring = smem_u32(room) + X_OFF + t * 4 * XB;
    long coming = first;
    int slot = 0;
    auto ahead = [&]() {  // the next row not yet under way
        if (coming < p.rows) {
#pragma unroll
            for (int k = 0; k < NCH; ++k)
                if (k * NEXT < left) {
                    copy_ahead<4 * DB>(ring + slot * STAGE + k * THREADS * 4 * DB, dy + k * NEXT * DB);
                    copy_ahead<4 * XB>(xring + slot * STAGE + k * THREADS * 4 * XB, x + k * NEXT * XB);
                }
        }
        cp_async_commit();  // an empty group keeps the count when there is no row left
        coming += step;
        dy += step * p.ldy;
        x += step * p.ldx;
        if (++slot == DEPTH) slot = 0;
    };
    if (AHEAD)
#pragma unroll
        for (int s = 0; s < DEPTH - 1; ++s) ahead();
    fetch(first < p.rows);
    char* dx = p.dx + first * p.lddx + first_c * (p.dx_wide ? 4 : 2);
    const char* add = p.add + first * p.lddx + first_c * (p.dx_wide ? 4 : 2);
    int stage = 0, turn = 0;
    for (long row = first; row < p.rows; row += step) {
        uint64_t h[NCH][2], g[NCH][2], red0 = 0, red1 = 0;
        const unsigned char *at = room + stage * STAGE + t * 4 * DB, *xat = room + stage * STAGE + X_OFF + t * 4 * XB;
        const float scale = next_scale, mean = next_mean, rstd = next_rstd;
        fetch(row + step < p.rows);
        if (AHEAD) {
            ahead();
            cp_async_wait<DEPTH - 1>();
            if (++stage == DEPTH) stage = 0;
        }
        const uint64_t minus = pair(-mean), r2 = pair(rstd);
#pragma unroll
        for (int k = 0; k < NCH; ++k) {  // dy * w, h and their sums
            if ((k * W + wid) * BLOCK >= p.dim) break;
            const int n = left - k * NEXT;
            float f[4] = {0.f, 0.f, 0.f, 0.f}, q[4] = {0.f, 0.f, 0.f, 0.f};
            if (AHEAD) {
                if (n > 0) {
                    read4<DB>(at + k * THREADS * 4 * DB, p.dy_half, f);
                    if (XB == 1) decode4(*reinterpret_cast<const uint32_t*>(xat + k * THREADS * 4), E4M3, q);
                    else read4<XB == 1 ? 2 : XB>(xat + k * THREADS * 4 * XB, p.x_half, q);
                }
            } else {
                load4_bytes<DB, false>(dy + k * NEXT * DB, p.dy_half, n, f);
                if (XB == 1) decode4(load_codes<false>(reinterpret_cast<const uint8_t*>(x) + k * NEXT, n), E4M3, q);
                else load4_bytes<XB == 1 ? 2 : XB, false>(x + k * NEXT * XB, p.x_half, n, q);
            }
            uint64_t d2[2], x2[2];
            pairs(f, d2);
            pairs(q, x2);
            const uint64_t s2 = XB == 1 ? pair(__shfl_sync(FULL_WARP, scale, k)) : 0;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint64_t d = XB == 1 ? fma2(x2[i], s2, minus) : add2(x2[i], minus);
                h[k][i] = mul2(d, r2);
                dw[k][i] = fma2(d2[i], h[k][i], dw[k][i]);
                db[k][i] = add2(db[k][i], d2[i]);
                g[k][i] = d2[i];
            }
            if (AHEAD) {
                g[k][0] = mul2(g[k][0], w2[k][0]);
                g[k][1] = mul2(g[k][1], w2[k][1]);
            } else if (p.w) {
                load4_const<false>(p.w + first_c + k * NEXT, n, f);
                pairs(f, w2[0]);
                g[k][0] = mul2(g[k][0], w2[0][0]);
                g[k][1] = mul2(g[k][1], w2[0][1]);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                red0 = add2(red0, g[k][i]);
                red1 = fma2(g[k][i], h[k][i], red1);
            }
        }
        if (!AHEAD) {
            dy += step * p.ldy;
            x += step * p.ldx;
        }
        const float2 red = row_sum2<W>(unpair(red0).x + unpair(red0).y, unpair(red1).x + unpair(red1).y,
                                       slots[turn][grp], wid, lane, 1 + grp);
        turn ^= 1;
        const uint64_t c1 = pair(-red.x * p.inv_dim), c2 = pair(-red.y * p.inv_dim);
#pragma unroll
        for (int k = 0; k < NCH; ++k) {
            if ((k * W + wid) * BLOCK >= p.dim) break;
            const int n = left - k * NEXT;
            uint64_t o[2] = {0, 0};
            float f[4];
            if (p.add) {
                if (p.dx_wide) load4_bytes<4, AHEAD>(add + k * NEXT * 4, false, n, f);
                else load4_bytes<2, AHEAD>(add + k * NEXT * 2, p.dx_half, n, f);
                pairs(f, o);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) o[i] = fma2(r2, fma2(h[k][i], c2, add2(g[k][i], c1)), o[i]);
            unpairs(o, f);
            if (p.dx_wide) store4_bytes<4, AHEAD>(dx + k * NEXT * 4, false, n, f);
            else store4_bytes<2, AHEAD>(dx + k * NEXT * 2, p.dx_half, n, f);
        }
        dx += step * p.lddx;
        add += step * p.lddx;
    }
    if (AHEAD) cp_async_wait<0>();
    __syncthreads();
    // the groups' sums, one group after the other
    float* sums = reinterpret_cast<float*>(room);
    for (int q = 0; q < G; ++q) {
        if (grp == q)
#pragma unroll
            for (int k = 0; k < NCH; ++k) {
                float a[4], b[4];
                unpairs(dw[k], a);
                unpairs(db[k], b);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int c = first_c + k * W * BLOCK + elem<AHEAD>(i);
                    if (c < p.dim) {
                        sums[c] = q == 0 ? a[i] : sums[c] + a[i];
                        sums[p.dim + c] = q == 0 ? b[i] : sums[p.dim + c] + b[i];
                    }
                }
            }
        __syncthreads();
    }
    pdl_trigger();
    float* out = p.part + (long)blockIdx.x * 2 * p.dim;
    for (int c = threadIdx.x; c < 2 * p.dim; c += THREADS) out[c] = sums[c];
}

template <int DB, int XB, int NCH>
constexpr int bwd_room() {
    constexpr int stage = BWD_WARPS * 32 * NCH * 4 * (DB + XB);
    return stage * BWD_DEPTH <= 160 * 1024 ? stage * BWD_DEPTH : 2 * stage;
}

// dw / db from nparts rows of partial sums: 32 columns a CTA, 32 lanes of parts each, added in a
// fixed order
__global__ void __launch_bounds__(1024) ln_sums_kernel(const float* part, int nparts, int dim, float* dw, float* db,
                                                       int accumulate) {
    __shared__ float s[32][33];
    const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    pdl_wait();
    float a = 0.f;
    if (c < 2 * dim)
#pragma unroll 8
        for (int q = slice; q < nparts; q += 32) a += part[(long)q * 2 * dim + c];
    s[slice][lane] = a;
    __syncthreads();
    if (slice || c >= 2 * dim) return;
#pragma unroll
    for (int q = 1; q < 32; ++q) a += s[q][lane];
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
    const long per = BWD_WARPS / bwd_warps(dim), need = (rows + per - 1) / per;
    const long sms = current_sm_count();
    return (int)(need < sms ? need : sms);
}

template <typename T, int W, int NCH, int G, bool VEC>
void launch_fwd(const FwdParams& p, cudaStream_t s) {
    // as many CTAs as run at once, each walking over rows
    static std::atomic<int> known[64];
    int dev = 0, per_sm = 0;
    const bool cached = cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64;
    if (cached) per_sm = known[dev].load(std::memory_order_relaxed);
    if (per_sm < 1) {
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, ln_fwd_kernel<T, W, NCH, G, VEC>, W * G * 32, 0) !=
                cudaSuccess || per_sm < 1) {
            cudaGetLastError();
            per_sm = 1;
        } else if (cached) {
            known[dev].store(per_sm, std::memory_order_relaxed);
        }
    }
    const long need = (p.rows + G - 1) / G, most = (long)per_sm * current_sm_count();
    ln_fwd_kernel<T, W, NCH, G, VEC><<<(unsigned)(need < most ? need : most), W * G * 32, 0, s>>>(p);
}

template <typename T, int W, int NCH, int G>
void launch_fwd(const FwdParams& p, bool vec, cudaStream_t s) {
    if (vec) launch_fwd<T, W, NCH, G, true>(p, s);
    else launch_fwd<T, W, NCH, G, false>(p, s);
}

// Up to eight blocks of 128 columns a warp: few exchanges between warps, and enough rows in flight
template <typename T>
void fwd_by_dim(const FwdParams& p, bool vec, cudaStream_t s) {
    if (p.dim <= 256) launch_fwd<T, 1, 2, 8>(p, vec, s);
    else if (p.dim <= 512) launch_fwd<T, 1, 4, 8>(p, vec, s);
    else if (p.dim <= 1024) launch_fwd<T, 2, 4, 4>(p, vec, s);
    else if (p.dim <= 1536) launch_fwd<T, 2, 6, 4>(p, vec, s);
    else if (p.dim <= 2048) launch_fwd<T, 2, 8, 4>(p, vec, s);
    else if (p.dim <= 4096) launch_fwd<T, 4, 8, 2>(p, vec, s);
    else launch_fwd<T, 8, 8, 1>(p, vec, s);
}

template <int DB, int XB, bool E4M3, int W, int NCH, bool AHEAD>
void launch_bwd(const BwdParams& p, int ctas, cudaStream_t s) {
    constexpr int most = 2 * NCH * BLOCK * W * (int)sizeof(float);  // sums of the widest row
    constexpr int smem = AHEAD && bwd_room<DB, XB, NCH>() > most ? bwd_room<DB, XB, NCH>() : most;
    static DeviceOnce once;
    once([] {
        cudaFuncSetAttribute(ln_bwd_kernel<DB, XB, E4M3, W, NCH, AHEAD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             smem);
    });
    ln_bwd_kernel<DB, XB, E4M3, W, NCH, AHEAD><<<ctas, BWD_WARPS * 32, smem, s>>>(p);
}

// three blocks a warp where they are enough (1536 columns on four warps): fewer registers, no idle block
template <int DB, int XB, bool E4M3, int W>
void launch_bwd(const BwdParams& p, bool vec, int ctas, cudaStream_t s) {
    if (!vec) launch_bwd<DB, XB, E4M3, W, BWD_NCH, false>(p, ctas, s);
    else if (p.dim <= 3 * W * BLOCK) launch_bwd<DB, XB, E4M3, W, 3, true>(p, ctas, s);
    else launch_bwd<DB, XB, E4M3, W, BWD_NCH, true>(p, ctas, s);
}

template <int DB, int XB, bool E4M3>
void bwd_by_dim(const BwdParams& p, bool vec, int ctas, cudaStream_t s) {
    switch (bwd_warps(p.dim)) {
        case 1: return launch_bwd<DB, XB, E4M3, 1>(p, vec, ctas, s);
        case 2: return launch_bwd<DB, XB, E4M3, 2>(p, vec, ctas, s);
        case 4: return launch_bwd<DB, XB, E4M3, 4>(p, vec, ctas, s);
        case 8: return launch_bwd<DB, XB, E4M3, 8>(p, vec, ctas, s);
        default: return launch_bwd<DB, XB, E4M3, 16>(p, vec, ctas, s);
    }
}

template <int DB>
void bwd_by_type(const BwdParams& p, int xb, bool e4m3, bool vec, int ctas, cudaStream_t s) {
    if (xb == 4) bwd_by_dim<DB, 4, false>(p, vec, ctas, s);
    else if (xb == 2) bwd_by_dim<DB, 2, false>(p, vec, ctas, s);
    else if (e4m3) bwd_by_dim<DB, 1, true>(p, vec, ctas, s);
    else bwd_by_dim<DB, 1, false>(p, vec, ctas, s);
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

size_t layernorm_train_bwd_space(long rows, long dim) {
    return (size_t)bwd_ctas(rows > 0 ? rows : 1, dim) * 2 * dim * sizeof(float);
}

void layernorm_train_bwd(const LnBwd& a, cudaStream_t s) {
    BwdParams p;
    p.rows = a.rows; p.ldy = a.dy.ld * op_bytes(a.dy.type); p.lddx = a.dx.ld * op_bytes(a.dx.type);
    p.dy = static_cast<const char*>(a.dy.p); p.dy_half = a.dy.type == OP_F16;
    p.x = a.x8.q ? reinterpret_cast<const char*>(a.x8.q) : static_cast<const char*>(a.x.p);
    p.ldx = a.x8.q ? a.x8.ldq : a.x.ld * op_bytes(a.x.type);
    p.x_half = a.x.type == OP_F16; p.scale = a.x8.scale; p.lds = a.x8.lds;
    p.add = static_cast<const char*>(a.add.p); p.dx = static_cast<char*>(const_cast<void*>(a.dx.p));
    p.dx_wide = a.dx.type == OP_F32; p.dx_half = a.dx.type == OP_F16; p.dim = a.dim;
    p.w = a.w; p.mean = a.mean; p.rstd = a.rstd; p.inv_dim = 1.0f / (float)a.dim; p.part = a.space;
    const bool vec = a.dim % 4 == 0 && vec4(a.dy) && vec4(a.x) && vec4(a.add) && vec4(a.dx) && vec4(a.x8) && vec4(a.w);
    const int ctas = a.rows > 0 ? bwd_ctas(a.rows, a.dim) : 0;
    if (ctas) {
        const int xb = a.x8.q ? 1 : op_bytes(a.x.type);
        if (op_bytes(a.dy.type) == 4) bwd_by_type<4>(p, xb, a.x8.e4m3, vec, ctas, s);
        else bwd_by_type<2>(p, xb, a.x8.e4m3, vec, ctas, s);
    }
    if (a.dw || a.db)
        launch_pdl(ln_sums_kernel, dim3((2 * a.dim + 31) / 32), dim3(1024), 0, s, (const float*)a.space, ctas, a.dim,
                   a.dw, a.db, a.accumulate ? 1 : 0);
}

}  // namespace act
