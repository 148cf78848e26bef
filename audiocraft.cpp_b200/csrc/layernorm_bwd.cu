// layernorm_bwd.cu -- layer norm whose weight and bias learn, backward: dx from dy and the input as it
// was or as its 8-bit checkpoint, and the sums over the rows that are the weight's and the bias's
// gradients.
//
// Every element is read once into registers, four columns a lane and up to NCH blocks of 128 columns a
// warp, by W warps a row.
// All statistics and sums are fp32.
// 24000 x 1536 with bf16 dy and dx and x in I8: 63 us with the sums over the CTAs, 2.9 TB/s (46% of HBM's
// rate), at 2.3 of 4 issues a cycle and a quarter of the warps, which is all that the sums' registers
// leave: a group waits for its row's two sums before it can write.
#include "layernorm.cuh"

namespace act {

namespace {

using namespace ln;

// A CTA's G row groups of W warps walk over rows; each lane keeps the sums dw and db of
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
// ahead, everything moves four elements at a time and w stays in registers.  Columns past the row's
// end read as x = 0 and dy = 0, so that they add nothing to any sum whatever their h is.
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
