// rank_ckpt8.cu -- the rank product that reads an 8-bit checkpoint: C[j][c] (+)= alpha * sum over
// rows t of U[t][j] * X[t][c], the lora_A gradient from a kept input.
//
// X is read once and the work per byte is small, so the kernel is bound by HBM as long as turning
// codes into tensor-core operands keeps up.  A CTA owns 128 or 256 columns of X (the rows of the MMA)
// and a slice of the rows t (the reduction), in blocks of 64:
//   warp 0     TMA: raw codes into a ring of 64-row blocks
//   warps 2, 3 U and the scales into the same ring (cp.async; loads to the converting warps' registers one
//              block ahead came too late: 24000 x 6144, rank 16, f16 U 94 us, so 70)
//   warps 8-15 codes * scale -> bf16 (4 or 7 significant bits times a power of two: exact down to bf16's
//              smallest step 2^-133) in the 128-byte-swizzled MN-major layout; the block's rows of U, cut
//              into bf16 pieces that add up to it (one for bf16, two for f16, three for fp32; bits below
//              2^-133 are cut off): both operands of the MMA have to be bf16, and the product keeps U
//   warp 1     tcgen05 MMAs, the pieces side by side as their columns (one reading of the X tile feeds all)
//   warps 4-7  the sums: the tensor cores cut each addition into the accumulator off below its last bit
//              (measured: a relative 2^-24 downwards per 16 rows, 5e-6 over 4000 rows), so the
//              accumulators are emptied into fp32 registers every 256 rows (two in turn where they fit)
// The slices of a column tile form a cluster and add their sums in order through distributed
// shared memory: no atomics, the same bits every time.
// 24000 x 6144 from E4M3 and I8: rank 16 with f16 U 70 us (2.2 TB/s) and 89 us, rank 64 with bf16 U 87 and
// 90 us, with fp32 U 104 and 112 us (shared memory and conversion take over from HBM).
#include <cuda.h>

#include <atomic>
#include <cstring>
#include <type_traits>

#include "ckpt8.cuh"
#include "slices.h"
#include "tc_common.cuh"

namespace act {

namespace {

using namespace c8;
using namespace tc;

constexpr int RK = 64;                   // rows t of a block
constexpr int RGROUP = 4;                // blocks between two emptyings of the accumulators
constexpr int RCONV = 8;                 // converting warps
constexpr int RROWS = RK / RCONV;        // rows of a block each takes
constexpr int RTHREADS = (8 + RCONV) * 32;
constexpr int RA_BYTES = 128 * RK * 2;   // bf16 operand of 128 columns
constexpr int RB_BOX = RK * 64 * 2;      // 64 columns of pieces
constexpr int RMAX_SPLIT = 16;           // cluster size, beyond the portable 8 by opt-in
constexpr int RNU = (RROWS * 8 + 31) / 32;  // units of 8 columns of U that a lane converts
constexpr int RSMEM_MAX = 232448;

// T: tiles of 128 columns per CTA; P: pieces of U, E: bytes of one of its values
template <int T, int P, int E>
struct RShape {
    static constexpr int RAW = T * 128 * RK;
    static constexpr int OP = T * RA_BYTES + P * RB_BOX;
    static constexpr int OPS = T == 2 ? 2 : 3;
    static constexpr int ACC = P * 64;                      // TMEM columns of a tile's accumulator
    static constexpr int BUFS = 2 * T * ACC <= 512 ? 2 : 1;  // of all tiles' accumulators
    static constexpr int TMEM = BUFS * T * ACC <= 128 ? 128 : BUFS * T * ACC <= 256 ? 256 : 512;
    static constexpr int U_BYTES = RCONV * 32 * RNU * 8 * E;  // U of a block
    static constexpr int SC_BYTES = T * RK * 4;               // its scales
    static constexpr int RAW_OFF = OPS * OP;
    static constexpr int FIT = (RSMEM_MAX - 2048 - RAW_OFF) / (RAW + U_BYTES + SC_BYTES);
    static constexpr int RAWS = FIT < 8 ? FIT : 8;
    static constexpr int U_OFF = RAW_OFF + RAWS * RAW;
    static constexpr int SC_OFF = U_OFF + RAWS * U_BYTES;
    static constexpr int BAR_OFF = SC_OFF + RAWS * SC_BYTES;
    static constexpr int NBARS = 2 * RAWS + 2 * OPS + 5;
    static constexpr int SMEM = BAR_OFF + 8 * NBARS + 16 + 1024 /*align*/;
    static constexpr int LD = T * 128 + 4;   // floats of a row of the sums in shared memory
    static_assert(RAWS >= 3 && SMEM <= RSMEM_MAX, "shared memory");
    static_assert(64 * LD * 4 <= RAW_OFF, "the sums take the operand ring's place");
};

struct RParams {
    int rows, nk, nb, nbp;  // nbp: nb rounded up to 16
    long cols;
    const void* u;
    int u_copy;  // bytes of a copy of U to shared memory: 16 or 8; 0: through registers
    long ldu;
    const float* scale;
    long lds;
    float alpha;
    float* c;
    long ldc;
    int c_vec, accumulate, splits;
    int* status;
};

struct RMaps {
    CUtensorMap x;
};

// B bytes, or zeros when !is (nothing is read then)
template <int B>
__device__ __forceinline__ void cp_async_to(uint32_t to, const void* from, bool is) {
    if (B == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(is ? 16 : 0)
                     : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(to), "l"(from), "n"(B), "r"(is ? B : 0)
                     : "memory");
}

__device__ __forceinline__ uint32_t pair_bf16(uint64_t v) {
    const float2 f = unpair(v);
    return pack_bf16(f.x, f.y);
}

// eight codes times s -> eight bf16
template <bool E4M3>
__device__ __forceinline__ uint4 codes_to_bf16(uint2 w, float s) {
    const uint64_t s2 = pair(s);
    uint32_t o[4];
    if (E4M3) {
        const uint32_t q[4] = {w.x & 0xffffu, w.x >> 16, w.y & 0xffffu, w.y >> 16};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2 h = __half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)q[i], __NV_E4M3));
            const float2 f = __half22float2(h);
            o[i] = pair_bf16(mul2(pair(f.x, f.y), s2));
        }
        return make_uint4(o[0], o[1], o[2], o[3]);
    }
    // q + 128 in the low byte of 2^23, less 2^23 + 128, times s: exact throughout
    const uint32_t x[2] = {w.x ^ 0x80808080u, w.y ^ 0x80808080u};
    const uint64_t bias = pair(-8388736.0f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t y = x[i >> 1];
        const int b = 2 * (i & 1);
        const float lo = __uint_as_float(__byte_perm(y, 0x4b000000u, 0x7650 + b));
        const float hi = __uint_as_float(__byte_perm(y, 0x4b000000u, 0x7651 + b));
        o[i] = pair_bf16(mul2(add2(pair(lo, hi), bias), s2));
    }
    // a zero byte of x is the code -128, NaN (a borrow may flag the byte above it too)
    const uint32_t z = ((x[0] - 0x01010101u) & ~x[0]) | ((x[1] - 0x01010101u) & ~x[1]);
    if (z & 0x80808080u)
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (((x[i >> 2] >> (8 * (i & 3))) & 0xffu) == 0) o[i >> 1] |= 0x7fc0u << (16 * (i & 1));
    return make_uint4(o[0], o[1], o[2], o[3]);
}

// Eight neighbouring values of a row of U as they lie in memory; `have` counts the columns from the
// first one (0: none), missing ones are 0.
template <typename U>
struct UnitOfU {
    static constexpr int W16 = 8 * sizeof(U) / 16;  // 16-byte words
    uint4 w[W16];
    __device__ __forceinline__ void load(const U* at, int have) {
        U e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = i < have ? at[i] : U(0.f);
        memcpy(w, e, sizeof(e));
    }
    // from global to shared memory in pieces of B bytes; word i of the unit lies at to + 512 i
    template <int B>
    static __device__ __forceinline__ void copy(uint32_t to, const U* at, int have) {
#pragma unroll
        for (int i = 0; i < 128 / B * (int)sizeof(U) / 16; ++i) {
            constexpr int V = B / (int)sizeof(U);
            const bool is = i * V < have;
            cp_async_to<B>(to + i * B / 16 * 512 + i * B % 16, at + (is ? i * V : 0), is);
        }
    }
    __device__ __forceinline__ void values(float v[8]) const {
        U e[8];
        memcpy(e, w, sizeof(e));
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_f32(e[i]);
    }
};

// bf16 pieces that hold all of a value of U
template <typename U>
struct Pieces {
    static constexpr int N = sizeof(U) == 4 ? 3 : std::is_same<U, f16>::value ? 2 : 1;
};

template <int T, bool E4M3, typename U>
__global__ void __launch_bounds__(RTHREADS, 1) rank_kernel(const __grid_constant__ RMaps maps, const RParams p) {
    constexpr int PIECES = Pieces<U>::N;
    typedef RShape<T, PIECES, sizeof(U)> S;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023) & ~1023u;
    unsigned char* smem = smem_raw + (base - raw);
    const uint32_t bars = base + S::BAR_OFF;
    auto raw_full = [&](int s) { return bars + 8 * s; };
    auto raw_empty = [&](int s) { return bars + 8 * (S::RAWS + s); };
    auto op_full = [&](int s) { return bars + 8 * (2 * S::RAWS + s); };
    auto op_empty = [&](int s) { return bars + 8 * (2 * S::RAWS + S::OPS + s); };
    auto acc_full = [&](int b) { return bars + 8 * (2 * S::RAWS + 2 * S::OPS + b); };
    auto acc_empty = [&](int b) { return bars + 8 * (2 * S::RAWS + 2 * S::OPS + 2 + b); };
    const uint32_t drained = bars + 8 * (2 * S::RAWS + 2 * S::OPS + 4);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + S::BAR_OFF + 8 * S::NBARS);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long c0 = (long)blockIdx.x * (T * 128);
    const int split = blockIdx.y;
    const int kb0 = (int)((long)p.nk * split / p.splits), kb1 = (int)((long)p.nk * (split + 1) / p.splits);

    if (threadIdx.x == 0) {
        prefetch_tmap(&maps.x);
        for (int s = 0; s < S::RAWS; ++s) {
            mbar_init(raw_full(s), 1 + 64);  // and every lane of warps 2 and 3
            mbar_init(raw_empty(s), RCONV);
        }
        for (int s = 0; s < S::OPS; ++s) {
            mbar_init(op_full(s), RCONV);
            mbar_init(op_empty(s), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(acc_full(b), 1);
            mbar_init(acc_empty(b), 4);
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

    // Launched with 128 registers a thread: 56 + 152 + 2 * 152 = 4 * 128.
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == 0 && lane == 0) {
            // -------------------------------------------------------- TMA
            int s = 0, issued = 0;
            uint32_t ph = 0;
            for (int kb = kb0; kb < kb1; ++kb, ++issued) {
                if (!mbar_wait_inline(raw_empty(s), ph ^ 1, p.status, 41)) break;
                mbar_expect_tx(raw_full(s), S::RAW);
                tma_load_2d(base + S::RAW_OFF + s * S::RAW, &maps.x, (int)c0, kb * RK, raw_full(s));
                if (++s == S::RAWS) { s = 0; ph ^= 1; }
            }
            drain_ring(raw_full(0), S::RAWS, issued);
        } else if (warp == 1 && lane == 0) {
            // -------------------------------------------------------- MMA
            // fp32 accumulator, bf16 operands (1), both MN-major, N >> 3, M >> 4
            const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 15) | (1u << 16) |
                                   ((uint32_t)((PIECES * p.nbp) >> 3) << 17) | (8u << 24);
            const uint64_t a_desc = smem_desc(base, 8192, 1024);
            const uint64_t b_desc = smem_desc(base + T * RA_BYTES, 8192, 1024);
            constexpr uint32_t step = 2048 >> 4;  // 16 rows of 128 bytes
            int s = 0, b = 0;
            uint32_t ph = 0, bph = 0;
            for (int kb = kb0; kb < kb1; ++kb) {
                const int in_group = (kb - kb0) % RGROUP;
                if (in_group == 0 && !mbar_wait_inline(acc_empty(b), bph ^ 1, p.status, 42)) break;
                if (!mbar_wait_inline(op_full(s), ph, p.status, 43)) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint64_t off = (uint64_t)((s * S::OP) >> 4);
#pragma unroll
                for (int t = 0; t < T; ++t) {
                    const uint64_t a = a_desc + off + (t * RA_BYTES >> 4), bb = b_desc + off;
#pragma unroll
                    for (int k = 0; k < RK / 16; ++k)
                        mma_f16(tmem + (b * T + t) * S::ACC, a + step * k, bb + step * k, idesc,
                                (in_group > 0 || k > 0) ? 1u : 0u);
                }
                mma_commit(op_empty(s));
                if (++s == S::OPS) { s = 0; ph ^= 1; }
                if (in_group == RGROUP - 1 || kb == kb1 - 1) {
                    mma_commit(acc_full(b));
                    if (++b == S::BUFS) { b = 0; bph ^= 1; }
                }
            }
            drain_mma(drained);
        } else if (warp >= 2) {
            // -------------------------------------------------------- U and scales
            // Copied as they are, each unit to where the lane that converts it reads it.
            constexpr int W16 = UnitOfU<U>::W16;
            const int w0 = (warp - 2) * (RCONV / 2);  // for converting warps w0 .. w0 + RCONV / 2 - 1
            const int units = p.nbp >> 3;
            int s = 0;
            uint32_t ph = 0;
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!__all_sync(FULL_WARP, mbar_wait_inline(raw_empty(s), ph ^ 1, p.status, 48))) break;
                const int t0 = kb * RK;
#pragma unroll
                for (int j = 0; j < T; ++j) {
                    const int e = ((warp - 2) * T + j) * 32 + lane, r = e % RK;
                    const long cb = c0 / BLOCK + e / RK;
                    const bool is = cb * BLOCK < p.cols && t0 + r < p.rows;
                    cp_async_to<4>(base + S::SC_OFF + s * S::SC_BYTES + 4 * e,
                                   is ? p.scale + cb * p.lds + t0 + r : p.scale, is);
                }
#pragma unroll
                for (int i = 0; i < RNU; ++i) {
                    const int q = lane + 32 * i, uj = q % units, ur = q / units;
                    if (ur >= RROWS || !p.u_copy) break;
                    const int have = p.nb - 8 * uj;
                    uint32_t to = base + S::U_OFF + s * S::U_BYTES + (w0 * RNU + i) * W16 * 512 + 16 * lane;
                    int t = t0 + w0 * RROWS + ur;
                    const U* at = static_cast<const U*>(p.u) + (long)t * p.ldu + 8 * uj;
#pragma unroll 1
                    for (int c = 0; c < RCONV / 2; ++c) {
                        const int n = t < p.rows && have > 0 ? have : 0;
                        const U* a = n ? at : static_cast<const U*>(p.u);
                        if (p.u_copy == 16) UnitOfU<U>::template copy<16>(to, a, n);
                        else UnitOfU<U>::template copy<8>(to, a, n);
                        t += RROWS;
                        at += RROWS * p.ldu;
                        to += RNU * W16 * 512;
                    }
                }
                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(raw_full(s)) : "memory");
                if (++s == S::RAWS) { s = 0; ph ^= 1; }
            }
            cp_async_wait_all();
        }
    } else if (warp < 8) {
        // ------------------------------------------------------------ sums
        asm volatile("setmaxnreg.inc.sync.aligned.u32 152;");
        const int quad = warp & 3;
        const uint32_t tl = tmem + ((uint32_t)(quad * 32) << 16);
        float sum[T][64];
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
            for (int i = 0; i < 64; ++i) sum[t][i] = 0.f;
        int b = 0;
        uint32_t bph = 0;
        bool ok = true;
        for (int kb = kb0; kb < kb1; kb += RGROUP) {
            if (!__all_sync(FULL_WARP, mbar_wait_inline(acc_full(b), bph, p.status, 44))) { ok = false; break; }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
            for (int t = 0; t < T; ++t)
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (16 * c < p.nbp) {
                        const uint32_t at = tl + (b * T + t) * S::ACC + 16 * c;
#pragma unroll
                        for (int q = PIECES - 1; q >= 0; --q) {  // the smallest piece first
                            uint32_t r[16];
                            tmem_ld16_start(at + q * p.nbp, r);
                            tmem_ld16_wait(r);
#pragma unroll
                            for (int i = 0; i < 16; ++i) sum[t][16 * c + i] += __uint_as_float(r[i]);
                        }
                    }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            if (lane == 0) mbar_arrive(acc_empty(b));
            if (++b == S::BUFS) { b = 0; bph ^= 1; }
        }
        if (ok) {  // every MMA is done: the operand ring is free
            float* part = reinterpret_cast<float*>(smem);
#pragma unroll
            for (int t = 0; t < T; ++t)
#pragma unroll
                for (int i = 0; i < 64; ++i)
                    if (i < p.nb) part[i * S::LD + t * 128 + quad * 32 + lane] = sum[t][i];
        }
    } else {
        // ------------------------------------------------------------ codes and U to bf16
        asm volatile("setmaxnreg.inc.sync.aligned.u32 152;");
        constexpr int LPR = 16 * T;        // lanes of a row (8 codes each)
        constexpr int RPP = 32 / LPR;      // rows of a pass
        const int cw = warp - 8, r0 = RROWS * cw;  // rows r0 .. r0 + RROWS - 1 of each block
        const int cl = lane % LPR, tile = cl >> 4, box = (cl >> 3) & 1, unit = cl & 7;
        // U: RROWS x nbp / 8 units of 8 columns, up to NU a lane
        constexpr int NU = RNU;
        const int units = p.nbp >> 3;
        bool has[NU];
        int ur[NU], have[NU];  // a unit's row in the warp's part and its columns that exist
        const U* from[NU];
        // where its pieces go in an operand slot: piece after piece, end to end
        uint32_t u_to[NU][PIECES];
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            const int q = lane + 32 * i, uj = q % units;
            ur[i] = q / units;
            has[i] = ur[i] < RROWS;
            have[i] = has[i] ? p.nb - 8 * uj : 0;
            from[i] = static_cast<const U*>(p.u) + (long)(r0 + ur[i]) * p.ldu + 8 * uj;
#pragma unroll
            for (int piece = 0; piece < PIECES; ++piece) {
                const int col8 = piece * units + uj;
                u_to[i][piece] = T * RA_BYTES + (col8 >> 3) * RB_BOX + q8_sw128(r0 + ur[i], col8 & 7);
            }
        }
        // Values at odd places are loaded by their own lane one block ahead: copies of 4 bytes keep warps 2
        // and 3 longer (22317 x 25 E4M3, fp32, rank 51: 37 us against 27).
        UnitOfU<U> un[NU];
        auto load = [&](int kb) {
#pragma unroll
            for (int i = 0; i < NU; ++i)
                un[i].load(from[i] + (long)kb * RK * p.ldu, kb * RK + r0 + ur[i] < p.rows ? have[i] : 0);
        };
        if (!p.u_copy && kb0 < kb1) load(kb0);
        int s = 0, o = 0;
        uint32_t ph = 0, oph = 0;
        for (int kb = kb0; kb < kb1; ++kb) {
            float u[NU][8];
            if (!p.u_copy) {
#pragma unroll
                for (int i = 0; i < NU; ++i) un[i].values(u[i]);
                if (kb + 1 < kb1) load(kb + 1);
            }
            // every lane waits (a lane that waited for its warp would cost the warp a detour); they agree
            const bool got = mbar_wait_inline(op_empty(o), oph ^ 1, p.status, 46) &&
                             mbar_wait_inline(raw_full(s), ph, p.status, 47);
            if (!__all_sync(FULL_WARP, got)) break;
            unsigned char* op = smem + o * S::OP;
            if (p.u_copy)
#pragma unroll
                for (int i = 0; i < NU; ++i)
#pragma unroll
                    for (int j = 0; j < UnitOfU<U>::W16; ++j)
                        un[i].w[j] = *reinterpret_cast<const uint4*>(
                            smem + S::U_OFF + s * S::U_BYTES + ((cw * NU + i) * UnitOfU<U>::W16 + j) * 512 + 16 * lane);
            const float* sc = reinterpret_cast<const float*>(smem + S::SC_OFF + s * S::SC_BYTES) + tile * RK + r0;
            const unsigned char* rw = smem + S::RAW_OFF + s * S::RAW;
            uint2 w[RROWS / RPP];
#pragma unroll
            for (int i = 0; i < RROWS / RPP; ++i)
                w[i] = *reinterpret_cast<const uint2*>(rw + (r0 + i * RPP + lane / LPR) * (T * 128) + 8 * cl);
#pragma unroll
            for (int i = 0; i < RROWS / RPP; ++i) {
                const int r = i * RPP + lane / LPR;
                *reinterpret_cast<uint4*>(op + tile * RA_BYTES + box * 8192 + q8_sw128(r0 + r, unit)) =
                    codes_to_bf16<E4M3>(w[i], sc[r]);
            }
            if (p.u_copy)
#pragma unroll
                for (int i = 0; i < NU; ++i) un[i].values(u[i]);
            __syncwarp();  // every lane has read the slot
            if (lane == 0) mbar_arrive(raw_empty(s));
            // The next piece of a value is its upper half-word (cut off, not rounded: three pieces hold all
            // 24 bits and none can overflow); what is left of it is exact.  Of an infinity nothing is left: one
            // test of a unit's largest value, 24000 x 6144 rank 64 with fp32 U 109 us before and 112 us with it
            // (taking NaN sums again at the end instead costs as much, and milliseconds where there are some).
#pragma unroll
            for (int i = 0; i < NU; ++i) {
                if (!has[i]) break;
                float top = 0.f;
                if (PIECES > 1)
#pragma unroll
                    for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(u[i][j]));
                const bool infinite = top == __int_as_float(0x7f800000);
#pragma unroll
                for (int piece = 0; piece < PIECES; ++piece) {
                    uint32_t h[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        h[j] = __byte_perm(__float_as_uint(u[i][2 * j]), __float_as_uint(u[i][2 * j + 1]), 0x7632);
                    *reinterpret_cast<uint4*>(op + u_to[i][piece]) = make_uint4(h[0], h[1], h[2], h[3]);
                    if (piece == 0 && infinite) {
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            u[i][j] = fabsf(u[i][j]) == __int_as_float(0x7f800000) ? 0.f :
                                u[i][j] - __uint_as_float(__float_as_uint(u[i][j]) & 0xffff0000u);
                    } else if (piece + 1 < PIECES)
#pragma unroll
                        for (int j = 0; j < 8; ++j) u[i][j] -= __uint_as_float(__float_as_uint(u[i][j]) & 0xffff0000u);
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(op_full(o));
            if (++s == S::RAWS) { s = 0; ph ^= 1; }
            if (++o == S::OPS) { o = 0; oph ^= 1; }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    // every warp has the launch's registers again for what all of them do from here on
    if (warp < 4) asm volatile("setmaxnreg.inc.sync.aligned.u32 128;");
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 128;");
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (warp == 0)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::TMEM));
    // every thread of every CTA of the cluster passes both barriers
    if (p.splits > 1) cluster_sync_all();
    const uint32_t part = base;
    const int rank = p.splits > 1 ? (int)cluster_ctarank() : 0;
    constexpr int Q = T * 32;  // float4 of a row
    const int items = p.nb * Q, i0 = (int)((long)items * rank / p.splits),
              i1 = (int)((long)items * (rank + 1) / p.splits);
    for (int i = i0 + threadIdx.x; i < i1; i += RTHREADS) {
        const int j = i / Q, f = i % Q * 4;
        const long c = c0 + f;
        if (c >= p.cols) continue;
        const uint32_t at = part + (uint32_t)(j * S::LD + f) * 4;
        float4 d[RMAX_SPLIT];  // all under way together
#pragma unroll
        for (int q = 0; q < RMAX_SPLIT; ++q)
            if (q < p.splits) d[q] = ld_dsmem_f4(p.splits > 1 ? map_cta(at, (uint32_t)q) : at);
        float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int q = 0; q < RMAX_SPLIT; ++q)  // slice order: the same sum whoever finished first
            if (q < p.splits) {
                v[0] += d[q].x; v[1] += d[q].y; v[2] += d[q].z; v[3] += d[q].w;
            }
        float* out = p.c + j * p.ldc + c;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] *= p.alpha;
        if (p.c_vec && c + 4 <= p.cols) {
            float4 w = make_float4(v[0], v[1], v[2], v[3]);
            if (p.accumulate) {
                const float4 old = *reinterpret_cast<const float4*>(out);
                w.x += old.x; w.y += old.y; w.z += old.z; w.w += old.w;
            }
            *reinterpret_cast<float4*>(out) = w;
        } else {
            for (int k = 0; k < 4 && c + k < p.cols; ++k) out[k] = p.accumulate ? out[k] + v[k] : v[k];
        }
    }
    if (p.splits > 1) cluster_sync_all();  // peers keep their sums until every reader is done
}

template <int T, bool E4M3, typename U>
void launch(const RankCkpt8& a, RParams p, cudaStream_t s) {
    typedef RShape<T, Pieces<U>::N, sizeof(U)> S;
    static DeviceOnce once;
    once([] {
        cudaFuncSetAttribute(rank_kernel<T, E4M3, U>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
    });
    const long tiles = (a.cols + T * 128 - 1) / (T * 128);
    // slices per tile: a round costs about eight blocks besides its own (start, join), without slices too
    static std::atomic<int> known[RMAX_SPLIT + 1][64];
    auto at_once = [](int n) { return clusters_at_once(rank_kernel<T, E4M3, U>, RTHREADS, S::SMEM, n, known[n]); };
    constexpr int JOIN = 8;
    const long room = at_once(1) > 1 ? at_once(1) : 1;
    p.splits = best_slices(tiles, p.nk, RMAX_SPLIT, JOIN, (tiles + room - 1) / room * (p.nk + JOIN), at_once);
    RMaps maps;
    tc_make_map_raw(&maps.x, a.x.q, false, a.rows, a.cols, a.x.ldq, T * 128, RK);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)tiles, (unsigned)p.splits, 1);
    cfg.blockDim = dim3(RTHREADS, 1, 1);
    cfg.dynamicSmemBytes = S::SMEM;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1;
    attr[0].val.clusterDim.y = (unsigned)p.splits;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, rank_kernel<T, E4M3, U>, maps, p);
}

template <int T, bool E4M3>
void launch(const RankCkpt8& a, const RParams& p, cudaStream_t s) {
    if (a.u.type == OP_F32) launch<T, E4M3, float>(a, p, s);
    else if (a.u.type == OP_F16) launch<T, E4M3, f16>(a, p, s);
    else launch<T, E4M3, __nv_bfloat16>(a, p, s);
}

}  // namespace

void rank_ckpt8(const RankCkpt8& a, cudaStream_t s) {
    if (!a.rows) {
        cudaMemset2DAsync(a.c, a.ldc * sizeof(float), 0, a.cols * sizeof(float), a.nb, s);
        return;
    }
    RParams p;
    p.rows = (int)a.rows; p.nk = (int)((a.rows + RK - 1) / RK); p.nb = a.nb; p.nbp = (a.nb + 15) / 16 * 16;
    p.cols = a.cols;
    p.u = a.u.p; p.ldu = a.u.ld;
    // the widest copy that base, stride and row length allow
    const int eb = op_bytes(a.u.type);
    p.u_copy = 0;
    for (int b = 16; b >= 8 && !p.u_copy; b >>= 1)
        if (a.nb * eb % b == 0 && a.u.ld * eb % b == 0 && reinterpret_cast<uintptr_t>(a.u.p) % b == 0) p.u_copy = b;
    p.scale = a.x.scale; p.lds = a.x.lds; p.alpha = a.alpha;
    p.c = a.c; p.ldc = a.ldc; p.c_vec = vec4(a.c) && a.ldc % 4 == 0 ? 1 : 0; p.accumulate = a.accumulate ? 1 : 0;
    p.splits = 1; p.status = a.status;
    // 256 columns a CTA halve the work on U per code, where that still leaves CTAs for most SMs
    const long wide = (a.cols + 255) / 256;
    if (wide * 8 >= current_sm_count()) a.x.e4m3 ? launch<2, true>(a, p, s) : launch<2, false>(a, p, s);
    else a.x.e4m3 ? launch<1, true>(a, p, s) : launch<1, false>(a, p, s);
}

}  // namespace act
