// gemm_f8.cu -- product of two E4M3 tensors with a scale for each block of 128:
//   Y[m][n] = sum over k-blocks b of sx[b][m] * sw[b][n / 128] * (sum over the block's k of X[m][k] W[n][k])
//
// The tensor cores take the codes as they are (tcgen05 kind::f8f6f4, fp32 accumulators in TMEM), one
// k-block of 128 at a time; a block's scales are constant over it for each (row, 128 columns), so
// its finished sum is multiplied by them once, in registers, on its way into the tile's sum.
//
// gemm_f8_kernel: one CTA per 128 x BN tile, persistent over tiles.  Warp 0 fills a ring of
// k-blocks by TMA (128-byte swizzle; rows and columns past the tensor's end read as zero), warp 2
// copies their scales, one thread of warp 1 issues four MMAs of 32 per k-block into one of two TMEM
// buffers, and eight warps take the buffers in turn: while the MMA of block i + 1 runs, they load
// block i from TMEM, multiply-add it into 128 x BN fp32 sums held in registers (two columns per
// instruction) and hand the buffer back.  A thread owns one row and half of the tile's columns;
// bias and the old value are added in fp32 before the one rounding.  A product of few tiles splits
// each tile's k-blocks over a cluster, whose CTAs add their sums in order.
// 24000 x 1536 x 6144 takes 210 us captured, 2160 TFLOP/s, and 248 us called in a loop (the power cap).
// The MMA alone takes 135 us, the loads alone 135 us, both without the adding 169 us: operand traffic and
// adding cost about the same beside the MMA.
//
// gemm_f8_small_kernel: up to 16 rows (a few tokens).  Bound by reading W once: a CTA owns 16 rows
// of W, its warps take turns with the k-blocks, and the codes go straight from global memory
// into mma.sync fragments: a lane loads 32 neighbouring codes of two rows of W and of its rows of
// X, which is a fixed permutation of the block's k that both operands share.  4 x 6144 x 1536: 4.6 us
// with W in L2, 6.5 us from HBM.
#include <cuda.h>

#include <atomic>

#include "ckpt8.cuh"
#include "slices.h"
#include "tc_common.cuh"

namespace act {

namespace {

using namespace c8;
using namespace tc;

constexpr int BM = 128, BK = 128;
constexpr int A_BYTES = BM * BK;
constexpr int NTHREADS = 384;  // four warps that feed, eight that add
constexpr int ADDERS = 8;
constexpr int SPLIT_LD = 128 + 4;  // floats of a row of a slice's sums
constexpr int MAX_SPLIT = 8;       // portable cluster size
// Scales of a k-block (128 of X, two of W) lie in a ring of their own: a slot is written when its
// stage is, at most STAGES blocks ahead of the MMAs, and read at most two blocks (the TMEM
// buffers) behind them, so that it is not overwritten before STAGES + 2 blocks have passed.
constexpr int SCALE_SLOTS = 8;
constexpr int SCALE_LD = BM + 4;  // floats
constexpr int SCALE_BYTES = SCALE_SLOTS * SCALE_LD * 4;
constexpr int TURN_LD = 17;  // floats of a row of 16 that a warp turns for rows of y that are not aligned
constexpr int TURN_BYTES = 32 * TURN_LD * 4;

// BN: columns of a tile
template <int BN>
struct Shape {
    static constexpr int STAGE = A_BYTES + BN * BK;
    static constexpr int STAGES = BN == 256 ? 4 : 6;
    static constexpr int HALF = BN / 2;  // columns of an adding warp
    static constexpr int SCALE_OFF = STAGES * STAGE;
    static constexpr int TURN_OFF = SCALE_OFF + SCALE_BYTES;
    static constexpr int BAR_OFF = TURN_OFF + ADDERS * TURN_BYTES;
    static constexpr int SMEM = BAR_OFF + 8 * (2 * STAGES + 5) + 16 + 1024 /*align*/;
    static constexpr int TMEM = 2 * BN;
    static_assert(STAGES + 2 <= SCALE_SLOTS, "a scale would be overwritten before it is read");
};

struct Maps {
    CUtensorMap x, w;
};

struct Params {
    long M, N, K;
    int nk;           // k-blocks
    int mt, nt;       // tiles
    int dm, dn;       // the grid's stride over them
    int splits;       // SPLIT: CTAs (a cluster) that share a tile's k-blocks
    const float *sx, *sw;
    long ldsx, ldsw;
    int sx_vec;       // X's scales move four at a time
    const float* bias;
    void* y;
    int y_type, accumulate;
    long ldy;
    int vec;          // rows of y move in whole sectors, bias four at a time
    int* status;
};

__device__ __forceinline__ float old_value(const Params& p, long at) {
    if (p.y_type == OP_F32) return static_cast<const float*>(p.y)[at];
    if (p.y_type == OP_F16) return to_f32(static_cast<const f16*>(p.y)[at]);
    return to_f32(static_cast<const __nv_bfloat16*>(p.y)[at]);
}
__device__ __forceinline__ void put_value(const Params& p, long at, float v) {
    if (p.y_type == OP_F32) static_cast<float*>(p.y)[at] = v;
    else if (p.y_type == OP_F16) static_cast<f16*>(p.y)[at] = from_f32<f16>(v);
    else static_cast<__nv_bfloat16*>(p.y)[at] = from_f32<__nv_bfloat16>(v);
}

// a whole 32-byte sector in one access
__device__ __forceinline__ void store_sector(void* p, const uint32_t w[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                 "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}
__device__ __forceinline__ void load_sector(const void* p, uint32_t w[8]) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                 : "l"(p)
                 : "memory");
}

// 16 columns n .. n + 15 of an aligned row (all of them exist): bias, old value, one rounding; at
// counts elements of y.  They move as whole 32-byte sectors (a thread's neighbours hold other rows).
__device__ __forceinline__ void put16(const Params& p, long at, long n, float v[16]) {
    if (p.bias)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const float4 b = __ldg(reinterpret_cast<const float4*>(p.bias + n + i));
            v[i] += b.x; v[i + 1] += b.y; v[i + 2] += b.z; v[i + 3] += b.w;
        }
    if (p.y_type == OP_F32) {
        float* y = static_cast<float*>(p.y) + at;
#pragma unroll
        for (int h = 0; h < 16; h += 8) {
            if (p.accumulate) {
                uint32_t o[8];
                load_sector(y + h, o);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[h + i] += __uint_as_float(o[i]);
            }
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(v[h + i]);
            store_sector(y + h, w);
        }
        return;
    }
    uint16_t* y = static_cast<uint16_t*>(p.y) + at;
    const bool half = p.y_type == OP_F16;
    uint32_t w[8];
    if (p.accumulate) {
        load_sector(y, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 f = half ? unpack_f16(w[i])
                                  : make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
            v[2 * i] += f.x;
            v[2 * i + 1] += f.y;
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        w[i] = half ? pack_f16(v[2 * i], v[2 * i + 1]) : pack_bf16(v[2 * i], v[2 * i + 1]);
    store_sector(y, w);
}

// A lane's column n of the 32 rows from m0 on, every other row of them, from a warp's turned 16 columns:
// bias, old value, one rounding.
__device__ __forceinline__ void put_column(const Params& p, long m0, long n, const float* turn) {
    const int lane = threadIdx.x & 31, first = lane >> 4;
    const int rows = p.M - m0 < 32 ? (int)(p.M - m0) : 32;
    const float add = p.bias ? __ldg(p.bias + n) : 0.f;
    const float* from = turn + first * TURN_LD + (lane & 15);
    const long at = (m0 + first) * p.ldy + n, step = 2 * p.ldy;
    if (p.accumulate) {
        for (int r = first; r < rows; r += 2, from += 2 * TURN_LD) {
            const long o = at + (r - first) / 2 * step;
            put_value(p, o, old_value(p, o) + (*from + add));
        }
    } else if (p.y_type == OP_F32) {
        float* y = static_cast<float*>(p.y) + at;
#pragma unroll 4
        for (int r = first; r < rows; r += 2, from += 2 * TURN_LD, y += step) *y = *from + add;
    } else {
        uint16_t* y = static_cast<uint16_t*>(p.y) + at;
        const bool half = p.y_type == OP_F16;
#pragma unroll 4
        for (int r = first; r < rows; r += 2, from += 2 * TURN_LD, y += step) {
            const float v = *from + add;
            *y = half ? __half_as_ushort(__float2half_rn(v)) : __bfloat16_as_ushort(__float2bfloat16_rn(v));
        }
    }
}

// the tiles of one CTA, column tiles first: CTAs that run together share rows of X
template <bool SPLIT>
struct Walk {
    int m, n;
    __device__ __forceinline__ explicit Walk(const Params& p) {
        const int first = SPLIT ? blockIdx.x / p.splits : blockIdx.x;
        m = first / p.nt;
        n = first % p.nt;
    }
    __device__ __forceinline__ bool any(const Params& p) const { return m < p.mt; }
    __device__ __forceinline__ void next(const Params& p) {
        if (SPLIT) {
            m = p.mt;
            return;
        }
        m += p.dm;
        n += p.dn;
        if (n >= p.nt) {
            n -= p.nt;
            ++m;
        }
    }
};

// SPLIT: a CTA has one tile, and its slice of the k-blocks
template <int BN, bool MN, bool SPLIT>
__global__ void __launch_bounds__(NTHREADS, 1) gemm_f8_kernel(const __grid_constant__ Maps maps, const Params p) {
    typedef Shape<BN> S;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023) & ~1023u;
    unsigned char* smem = smem_raw + (base - raw);
    const uint32_t bars = base + S::BAR_OFF;
    auto full_bar = [&](int s) { return bars + 8 * s; };
    auto empty_bar = [&](int s) { return bars + 8 * (S::STAGES + s); };
    auto tfull = [&](int b) { return bars + 8 * (2 * S::STAGES + b); };
    auto tempty = [&](int b) { return bars + 8 * (2 * S::STAGES + 2 + b); };
    const uint32_t drained = bars + 8 * (2 * S::STAGES + 4);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + S::BAR_OFF + 8 * (2 * S::STAGES + 5));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        prefetch_tmap(&maps.x);
        prefetch_tmap(&maps.w);
        for (int s = 0; s < S::STAGES; ++s) {
            mbar_init(full_bar(s), 1 + 32);  // the tiles' bytes and the lanes that copy the scales
            mbar_init(empty_bar(s), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(tfull(b), 1);
            mbar_init(tempty(b), ADDERS);
        }
        mbar_init(drained, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(S::TMEM));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot;
    const int rank = SPLIT ? (int)cluster_ctarank() : 0;
    const int kb0 = SPLIT ? (int)((long)p.nk * rank / p.splits) : 0;
    const int kb1 = SPLIT ? (int)((long)p.nk * (rank + 1) / p.splits) : p.nk;

    // Registers: the four feeding warps give theirs to the eight that hold the sums (launched with
    // 168 each: 128 * 56 + 256 * 224 = 384 * 168).
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == 0 && lane == 0) {
            // -------------------------------------------------------- TMA
            int s = 0;
            uint32_t ph = 0;
            long issued = 0;
            bool ok = true;
            for (Walk<SPLIT> t(p); ok && t.any(p); t.next(p)) {
                const int m0 = t.m * BM, n0 = t.n * BN;
                for (int kb = kb0; kb < kb1; ++kb, ++issued) {
                    if (!mbar_wait_inline(empty_bar(s), ph ^ 1, p.status, 31)) { ok = false; break; }
                    const uint32_t sa = base + s * S::STAGE, sb = sa + A_BYTES;
                    mbar_expect_tx(full_bar(s), S::STAGE);
                    tma_load_2d(sa, &maps.x, kb * BK, m0, full_bar(s));
                    if (MN) {  // [K][N]: a box of 128 (n) x 128 (k) per 128 columns
#pragma unroll
                        for (int h = 0; h < BN / 128; ++h)
                            tma_load_2d(sb + h * 16384, &maps.w, n0 + 128 * h, kb * BK, full_bar(s));
                    } else {
                        tma_load_2d(sb, &maps.w, kb * BK, n0, full_bar(s));
                    }
                    if (++s == S::STAGES) { s = 0; ph ^= 1; }
                }
            }
            drain_ring(full_bar(0), S::STAGES, issued);
        } else if (warp == 2) {
            // -------------------------------------------------------- scales
            int s = 0, slot = 0;
            uint32_t ph = 0;
            bool ok = true;
            const uint32_t ring = base + S::SCALE_OFF;
            for (Walk<SPLIT> t(p); ok && t.any(p); t.next(p)) {
                // rows 4 lane .. 4 lane + 3 of X, and (lanes 0, 1) 128 columns of W each
                const long m = (long)t.m * BM + 4 * lane, n = (long)t.n * BN + 128 * lane;
                const bool whole = p.sx_vec && m + 4 <= p.M, w = lane < BN / 128 && n < p.N;
                const float* sx = p.sx + (long)kb0 * p.ldsx + m;
                // W's scales: [k-block][n-block], or [n-block][k-block] of a weight stored [K][N]
                const float* sw = p.sw + (w ? (MN ? n / 128 * p.ldsw : n / 128) : 0) + (long)kb0 * (MN ? 1 : p.ldsw);
                for (int kb = kb0; kb < kb1; ++kb) {
                    if (!__all_sync(FULL_WARP, mbar_wait_inline(empty_bar(s), ph ^ 1, p.status, 35))) { ok = false; break; }
                    const uint32_t to = ring + slot * SCALE_LD * 4;
                    if (whole) {
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + 16 * lane), "l"(sx) : "memory");
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (m + i < p.M)
                                asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to + 16 * lane + 4 * i),
                                             "l"(sx + i) : "memory");
                    }
                    if (w)
                        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to + 4 * (BM + lane)), "l"(sw)
                                     : "memory");
                    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(full_bar(s)) : "memory");
                    sx += p.ldsx;
                    sw += MN ? 1 : p.ldsw;
                    if (++slot == SCALE_SLOTS) slot = 0;
                    if (++s == S::STAGES) { s = 0; ph ^= 1; }
                }
            }
            cp_async_wait_all();
        } else if (warp == 1 && lane == 0) {
            // -------------------------------------------------------- MMA
            // fp32 accumulator (bit 4), E4M3 operands (0), B's major, N >> 3, M >> 4
            const uint32_t idesc = (1u << 4) | ((uint32_t)MN << 16) | ((uint32_t)(BN >> 3) << 17) |
                                   ((uint32_t)(BM >> 4) << 24);
            const uint64_t a_desc = smem_desc(base, 16, 1024);
            const uint64_t b_desc = MN ? smem_desc(base + A_BYTES, 16384, 1024) : smem_desc(base + A_BYTES, 16, 1024);
            constexpr uint32_t b_step = (MN ? 32 * 128 : 32) >> 4;  // 32 of k: rows of 128 bytes, or bytes of a row
            int s = 0, b = 0;
            uint32_t ph = 0, bph = 0;
            bool ok = true;
            for (Walk<SPLIT> t(p); ok && t.any(p); t.next(p)) {
                for (int kb = kb0; kb < kb1; ++kb) {
                    if (!mbar_wait_inline(tempty(b), bph ^ 1, p.status, 32) ||
                        !mbar_wait_inline(full_bar(s), ph, p.status, 33)) {
                        ok = false;
                        break;
                    }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint64_t off = (uint64_t)((s * S::STAGE) >> 4);
#pragma unroll
                    for (int k = 0; k < BK / 32; ++k)
                        mma_f8(tmem + b * BN, a_desc + off + 2 * k, b_desc + off + b_step * k, idesc, k > 0);
                    mma_commit(empty_bar(s));
                    mma_commit(tfull(b));
                    if (++s == S::STAGES) { s = 0; ph ^= 1; }
                    b ^= 1;
                    if (b == 0) bph ^= 1;
                }
            }
            drain_mma(drained);
        }
    } else {
        // ------------------------------------------------------------ adding warps
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        const int quad = warp & 3, half = (warp - 4) >> 2;
        const uint32_t tcol = tmem + ((uint32_t)(quad * 32) << 16) + half * S::HALF;
        const float* const scales = reinterpret_cast<const float*>(smem + S::SCALE_OFF);
        int slot = 0;
        int b = 0;
        uint32_t bph = 0;
        bool ok = true;
        for (Walk<SPLIT> w(p); ok && w.any(p); w.next(p)) {
            const long m0 = (long)w.m * BM + quad * 32, n0 = (long)w.n * BN + half * S::HALF;
            uint64_t acc[S::HALF / 2];
#pragma unroll
            for (int i = 0; i < S::HALF / 2; ++i) acc[i] = 0;
            for (int kb = kb0; kb < kb1; ++kb) {
                // every lane waits (a lane that waited for its warp would cost the warp a detour); they agree
                if (!__all_sync(FULL_WARP, mbar_wait_inline(tfull(b), bph, p.status, 34))) { ok = false; break; }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const float* at = scales + slot * SCALE_LD;
                const uint64_t sc = pair(at[quad * 32 + lane] * at[BM + (BN == 256 ? half : 0)]);
                if (++slot == SCALE_SLOTS) slot = 0;
                uint32_t r[2][16];
                tmem_ld16_start(tcol + b * BN, r[0]);
#pragma unroll
                for (int c = 0; c < S::HALF / 16; ++c) {
                    tmem_ld16_wait(r[c & 1]);
                    if (c + 1 < S::HALF / 16) {
                        tmem_ld16_start(tcol + b * BN + 16 * (c + 1), r[(c + 1) & 1]);
                    } else {  // all of this warp's part is read: hand the buffer back
                        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                        if (lane == 0) mbar_arrive(tempty(b));
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        acc[8 * c + i] = fma2(pair(__uint_as_float(r[c & 1][2 * i]), __uint_as_float(r[c & 1][2 * i + 1])),
                                              sc, acc[8 * c + i]);
                }
                b ^= 1;
                if (b == 0) bph ^= 1;
            }
            if (!ok) break;
            if (SPLIT) {  // this slice's sums, where the operand ring was: every MMA that read it is done
                float* to = reinterpret_cast<float*>(smem) + (quad * 32 + lane) * SPLIT_LD + half * S::HALF;
#pragma unroll
                for (int i = 0; i < S::HALF / 4; ++i) {
                    const float2 u = unpair(acc[2 * i]), v = unpair(acc[2 * i + 1]);
                    *reinterpret_cast<float4*>(to + 4 * i) = make_float4(u.x, u.y, v.x, v.y);
                }
                break;
            }
            // epilogue, 16 columns at a time: a row per thread where its pieces are whole sectors; else the
            // warp turns its 32 rows in shared memory and writes two of them at a time
            const long m = m0 + lane;
            float* turn = reinterpret_cast<float*>(smem + S::TURN_OFF + (warp - 4) * TURN_BYTES);
#pragma unroll
            for (int c = 0; c < S::HALF / 16; ++c) {
                const long n = n0 + 16 * c;
                float v[16];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float2 f = unpair(acc[8 * c + i]);
                    v[2 * i] = f.x;
                    v[2 * i + 1] = f.y;
                }
                if (p.vec && n + 16 <= p.N) {
                    if (m < p.M) put16(p, m * p.ldy + n, n, v);
                } else if (n < p.N) {
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 16; ++i) turn[lane * TURN_LD + i] = v[i];
                    __syncwarp();
                    if (n + (lane & 15) < p.N) put_column(p, m0, n + (lane & 15), turn);
                }
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (warp == 0)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::TMEM));
    if (SPLIT) {
        // every warp has the launch's registers again for what all of them do from here on
        if (warp < 4) asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
        else asm volatile("setmaxnreg.dec.sync.aligned.u32 168;");
        // every thread of every CTA of the cluster passes both barriers
        cluster_sync_all();
        const Walk<SPLIT> w(p);
        constexpr int G = BN / 4;  // groups of 4 columns of a row
        const int r0 = BM * rank / p.splits, r1 = BM * (rank + 1) / p.splits;
        for (int i = threadIdx.x; i < (r1 - r0) * G; i += NTHREADS) {
            const int r = r0 + i / G, c = i % G * 4;
            const long m = (long)w.m * BM + r, n = (long)w.n * BN + c;
            if (m >= p.M || n >= p.N) continue;
            const uint32_t at = base + (uint32_t)(r * SPLIT_LD + c) * 4;
            float4 d[MAX_SPLIT];  // all under way together
#pragma unroll
            for (int q = 0; q < MAX_SPLIT; ++q)
                if (q < p.splits) d[q] = ld_dsmem_f4(map_cta(at, (uint32_t)q));
            float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int q = 0; q < MAX_SPLIT; ++q)  // slice order: the same sum whoever finished first
                if (q < p.splits) {
                    v[0] += d[q].x; v[1] += d[q].y; v[2] += d[q].z; v[3] += d[q].w;
                }
            const long o = m * p.ldy + n;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (n + j < p.N) {
                    const float s = v[j] + (p.bias ? __ldg(p.bias + n + j) : 0.f);
                    put_value(p, o + j, p.accumulate ? old_value(p, o + j) + s : s);
                }
        }
        cluster_sync_all();  // peers keep their sums until every reader is done
    }
}

// ---------------------------------------------------------------------------------------
constexpr int SM_ROWS = 16;   // rows of W a CTA owns
constexpr int SM_MAX_M = 16;

__device__ __forceinline__ void mma_sync_e4m3(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 32 codes from k on (16-byte aligned); codes at or past K read as 0
__device__ __forceinline__ void load32(const uint8_t* row, long k, long K, bool in, uint32_t r[8]) {
    uint4 v[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
#pragma unroll
    for (int h = 0; h < 2; ++h)
        if (in && k + 16 * h < K) v[h] = *reinterpret_cast<const uint4*>(row + k + 16 * h);
    const uint32_t w[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = w[i];
    if (k + 32 > K)  // the row's end: what follows it in memory is anyone's
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const long left = K - (k + 4 * i);
            r[i] = left >= 4 ? r[i] : left > 0 ? r[i] & (0xffffffffu >> (32 - 8 * (int)left)) : 0u;
        }
}

// what a lane needs of a k-block: codes of two rows of W and MT rows of X, and the products of scales
template <int MT>
struct SmallBlock {
    uint32_t a[2][8], b[MT][8];
    float s[MT][2];
    __device__ __forceinline__ void load(const uint8_t* x, long ldx, const uint8_t* w, long ldw, const Params& p, long n,
                                         int g, int t, int kb) {
        const long k = (long)kb * BK + 32 * t;
        load32(w, k, p.K, n < p.N, a[0]);
        load32(w + 8 * ldw, k, p.K, n + 8 < p.N, a[1]);
        const float sw = p.sw[(long)kb * p.ldsw + n / 128];
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            load32(x + 8 * j * ldx, k, p.K, 8 * j + g < p.M, b[j]);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int m = 8 * j + 2 * t + c;
                s[j][c] = m < p.M ? sw * p.sx[(long)kb * p.ldsx + m] : 0.f;
            }
        }
    }
};

// MT groups of eight rows of X; WARPS share the k-blocks.  A warp has more than one block's loads under
// way: the kernel is a chain of HBM latencies otherwise.
template <int MT, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) gemm_f8_small_kernel(const uint8_t* x, long ldx, const uint8_t* w,
                                                                   long ldw, const Params p) {
    __shared__ float part[WARPS][8 * MT][SM_ROWS + 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const long n0 = (long)blockIdx.x * SM_ROWS, n = n0 + g;
    x += g * ldx;
    w += n * ldw;
    float acc[MT][4] = {};
    auto multiply = [&](const SmallBlock<MT>& now) {
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            float d[4] = {};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t f[4] = {now.a[0][2 * i], now.a[1][2 * i], now.a[0][2 * i + 1], now.a[1][2 * i + 1]};
                mma_sync_e4m3(d, f, now.b[j][2 * i], now.b[j][2 * i + 1]);
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[j][c] = fmaf(d[c], now.s[j][c & 1], acc[j][c]);
        }
    };
    if (MT == 1) {
        SmallBlock<MT> next;
        if (warp < p.nk) next.load(x, ldx, w, ldw, p, n, g, t, warp);
        for (int kb = warp; kb < p.nk; kb += WARPS) {
            const SmallBlock<MT> now = next;
            if (kb + WARPS < p.nk) next.load(x, ldx, w, ldw, p, n, g, t, kb + WARPS);
            multiply(now);
        }
    } else {  // two blocks at a time: a third would cost the registers that let all CTAs run at once
#pragma unroll 2
        for (int kb = warp; kb < p.nk; kb += WARPS) {
            SmallBlock<MT> now;
            now.load(x, ldx, w, ldw, p, n, g, t, kb);
            multiply(now);
        }
    }
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) part[warp][8 * j + 2 * t + (c & 1)][g + 8 * (c >> 1)] = acc[j][c];
    __syncthreads();
    for (int i = threadIdx.x; i < 8 * MT * SM_ROWS; i += WARPS * 32) {
        const int m = i / SM_ROWS, r = i % SM_ROWS;
        if (m >= p.M || n0 + r >= p.N) continue;
        float v = 0.f;
#pragma unroll
        for (int q = 0; q < WARPS; ++q) v += part[q][m][r];
        if (p.bias) v += p.bias[n0 + r];
        const long at = m * p.ldy + n0 + r;
        put_value(p, at, p.accumulate ? old_value(p, at) + v : v);
    }
}

template <int MT, int WARPS>
void launch_small(const GemmF8& a, const Params& p, cudaStream_t s) {
    gemm_f8_small_kernel<MT, WARPS><<<(unsigned)((a.N + SM_ROWS - 1) / SM_ROWS), WARPS * 32, 0, s>>>(
        a.x.q, a.x.ldq, a.w.q, a.w.ldq, p);
}

template <int BN, bool MN, bool SPLIT>
void launch(const GemmF8& a, Params p, cudaStream_t s) {
    typedef Shape<BN> S;
    static_assert(!SPLIT || (BN == 128 && BM * SPLIT_LD * 4 <= S::STAGES * S::STAGE),
                  "a slice's sums take the ring's place");
    static DeviceOnce once;
    once([] {
        cudaFuncSetAttribute(gemm_f8_kernel<BN, MN, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
    });
    Maps maps;
    tc_make_map_u8(&maps.x, a.x.q, a.M, a.K, a.x.ldq, BK, BM);
    if (MN) tc_make_map_u8(&maps.w, a.w.q, a.K, a.N, a.w.ldq, 128, BK);
    else tc_make_map_u8(&maps.w, a.w.q, a.N, a.K, a.w.ldq, BK, BN);
    p.mt = (int)((a.M + BM - 1) / BM);
    p.nt = (int)((a.N + BN - 1) / BN);
    const long tiles = (long)p.mt * p.nt, sms = current_sm_count();
    const int ctas = SPLIT ? (int)tiles * p.splits : (int)(tiles < sms ? tiles : sms);
    p.dm = ctas / p.nt;
    p.dn = ctas % p.nt;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas, 1, 1);
    cfg.blockDim = dim3(NTHREADS, 1, 1);
    cfg.dynamicSmemBytes = S::SMEM;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = SPLIT ? (unsigned)p.splits : 1;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, gemm_f8_kernel<BN, MN, SPLIT>, maps, p);
}

template <int BN, bool SPLIT>
void launch(const GemmF8& a, const Params& p, cudaStream_t s) {
    if (a.w_mn) launch<BN, true, SPLIT>(a, p, s);
    else launch<BN, false, SPLIT>(a, p, s);
}

// CTAs per tile for a product of tiles that all run at once: joining the slices costs about as long as
// twelve k-blocks
template <bool MN>
int best_split(long tiles, int nk) {
    static std::atomic<int> known[MAX_SPLIT + 1][64];
    return best_slices(tiles, nk, MAX_SPLIT, 12, nk, [](int n) {
        return clusters_at_once(gemm_f8_kernel<128, MN, true>, NTHREADS, Shape<128>::SMEM, n, known[n]);
    });
}

}  // namespace

void gemm_f8(const GemmF8& a, cudaStream_t s) {
    Params p;
    p.M = a.M; p.N = a.N; p.K = a.K; p.nk = (int)((a.K + BK - 1) / BK);
    p.sx = a.x.scale; p.sw = a.w.scale; p.ldsx = a.x.lds; p.ldsw = a.w.lds;
    p.sx_vec = vec4(a.x.scale) && a.x.lds % 4 == 0;
    p.bias = a.bias; p.y = const_cast<void*>(a.y.p); p.y_type = a.y.type; p.accumulate = a.accumulate ? 1 : 0;
    p.ldy = a.y.ld; p.status = a.status;
    p.vec = a.y.ld * op_bytes(a.y.type) % 32 == 0 && reinterpret_cast<uintptr_t>(a.y.p) % 32 == 0 && vec4(a.bias);
    p.mt = p.nt = p.dm = p.dn = 0;
    p.splits = 1;
    // A few rows: at 16 x 6144 x 1536 6.3 us against 8.6 us on a mostly empty tensor-core tile
    if (a.M <= SM_MAX_M && !a.w_mn) {
        // as many warps as leave each one or two k-blocks, as far as registers let all CTAs run at once
        if (a.M <= 8) p.nk > 16 ? launch_small<1, 16>(a, p, s) : launch_small<1, 8>(a, p, s);
        else p.nk > 16 ? launch_small<2, 8>(a, p, s) : launch_small<2, 4>(a, p, s);
        return;
    }
    const long mt = (a.M + BM - 1) / BM, sms = current_sm_count(), narrow = mt * ((a.N + 127) / 128);
    if (narrow < sms) {
        p.splits = a.w_mn ? best_split<true>(narrow, p.nk) : best_split<false>(narrow, p.nk);
        if (p.splits > 1) return launch<128, true>(a, p, s);
    }
    // 256-wide tiles unless 128-wide ones finish in fewer column-rounds over the SMs
    auto cost = [&](long bn) { return (mt * ((a.N + bn - 1) / bn) + sms - 1) / sms * bn; };
    if (cost(128) < cost(256)) launch<128, false>(a, p, s);
    else launch<256, false>(a, p, s);
}

}  // namespace act
