// ckpt8.cu -- activations put away in 8 bits and read back, alone and inside the GELU's forward
// and backward passes.
//
// Every kernel here is one pass over its tensors: store reads 4 or 2 bytes an element and writes 1 (+ 4
// bytes a block), load the reverse; the GELU's forward reads 2 and writes 2 + 1, its backward reads
// 2 + 1 and writes 2 (16-bit types).  Store and load are bound by HBM.  GELU is short of both limits,
// 77% of HBM's rate and 2.6 to 2.7 of 4 issues a cycle at a third of the warps: chains of dependent
// arithmetic in few warps.  A warp takes one block of 128 columns and RPW neighbouring rows of it at a
// time, with the next rows' loads under way: a block's maximum is one warp reduction, and the rows'
// scales, which lie next to each other (block-major), leave as one store.  GELU forward and backward of
// 12000 x 6144 bf16 with E4M3 checkpoint: 149 us, 5.0 TB/s (167 us called in a loop); store and load of
// 6144 x 1536 fp32 in 128 x 128 blocks: 14.8 us.
#include <type_traits>

#include "ckpt8.cuh"

namespace act {

namespace {

using namespace c8;

constexpr int RPW = 4;        // rows of a block column a warp holds at a time
constexpr int THREADS = 256;

// A warp's block column and its first row group; warps beyond the last whole set of block
// columns have none
struct Place {
    int chunk, n;         // block column; columns of the row from the lane's first one
    long col, row, step;  // the lane's first column, first row, rows between two groups of this warp
    bool any;
};
template <bool VEC>
__device__ __forceinline__ Place place(long cols) {
    const unsigned warp = blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5), nwarps = gridDim.x * (THREADS / 32);
    const unsigned chunks = (unsigned)((cols + BLOCK - 1) / BLOCK), lanes = nwarps / chunks;
    Place p;
    p.chunk = (int)(warp % chunks);
    p.row = (long)(warp / chunks) * RPW;
    p.step = (long)lanes * RPW;
    p.any = warp / chunks < lanes;
    p.col = (long)p.chunk * BLOCK + first_col<VEC>(threadIdx.x & 31);
    p.n = cols - p.col < BLOCK ? (int)(cols - p.col) : BLOCK;
    return p;
}

// body(place, held, row, rows, whole) for each of the warp's groups of up to RPW rows; `held` is what
// fetch(place, held, row, rows, whole) has loaded of them, one group ahead of its use.  `whole` (a
// type) says that all RPW rows exist, which saves the tests.
template <bool VEC, typename Held, typename Fetch, typename Body>
__device__ __forceinline__ void each_group(long rows, long cols, Fetch&& fetch, Body&& body) {
    const Place p = place<VEC>(cols);
    if (!p.any || p.row >= rows) return;
    Held next;
    long row = p.row;
    auto get = [&](long r) {
        if (r + RPW <= rows) fetch(p, next, r, RPW, std::true_type());
        else if (r < rows) fetch(p, next, r, (int)(rows - r), std::false_type());
    };
    get(row);
    for (; row + RPW <= rows; row += p.step) {
        const Held held = next;
        get(row + p.step);
        body(p, held, row, RPW, std::true_type());
    }
    if (row < rows) body(p, next, row, (int)(rows - row), std::false_type());
}

// the scales of up to RPW rows: lane r holds row r's
__device__ __forceinline__ void store_scales(const Q8& t, int chunk, long row, int nr, const uint32_t* s) {
    const int lane = threadIdx.x & 31;
    uint32_t mine = s[0];
#pragma unroll
    for (int r = 1; r < RPW; ++r) mine = lane == r ? s[r] : mine;
    if (lane < nr) t.scale[(long)chunk * t.lds + row + lane] = __uint_as_float(mine);
}

// v: RPW rows of a block, -> codes and scales
template <bool VEC, bool WHOLE>
__device__ __forceinline__ void store_rows(const Q8& t, const Place& p, long row, int nr, const float (*v)[4],
                                           bool e4m3) {
    uint32_t s[RPW], top[RPW], most = 0;
    uint8_t* q = t.q + row * t.ldq + p.col;
#pragma unroll
    for (int r = 0; r < RPW; ++r) {
        top[r] = __reduce_max_sync(FULL_WARP, largest(v[r]));
        most = max(most, top[r]);
    }
    if (most > limit_bits(e4m3)) {  // one test for all rows: something is beyond the limit or not finite
#pragma unroll
        for (int r = 0; r < RPW; ++r) {
            float w[4] = {v[r][0], v[r][1], v[r][2], v[r][3]};
            limit4(w, e4m3);
            s[r] = scale_bits(__reduce_max_sync(FULL_WARP, largest_finite(w)), e4m3);
            store_codes<VEC>(q + r * t.ldq, WHOLE || r < nr ? p.n : 0, encode4(w, inverse_pow2(s[r]), e4m3, true));
        }
    } else {
#pragma unroll
        for (int r = 0; r < RPW; ++r) {
            s[r] = scale_bits(top[r], e4m3);
            store_codes<VEC>(q + r * t.ldq, WHOLE || r < nr ? p.n : 0, encode4(v[r], inverse_pow2(s[r]), e4m3, false));
        }
    }
    store_scales(t, p.chunk, row, nr, s);
}

template <typename T, bool VEC>
struct HeldRows {
    Raw4<T, VEC> x[RPW];
    template <bool WHOLE>
    __device__ __forceinline__ void load(const T* at, long ld, int n, int nr) {
#pragma unroll
        for (int r = 0; r < RPW; ++r) x[r].load(at + r * ld, WHOLE || r < nr ? n : 0);
    }
};

template <typename T, bool VEC, bool E4M3>
__global__ void __launch_bounds__(THREADS) store_kernel(const T* x, long ldx, long rows, long cols, Q8 out) {
    typedef HeldRows<T, VEC> Held;
    each_group<VEC, Held>(
        rows, cols,
        [&](const Place& p, Held& h, long row, int nr, auto whole) {
            h.template load<decltype(whole)::value>(x + row * ldx + p.col, ldx, p.n, nr);
        },
        [&](const Place& p, const Held& h, long row, int nr, auto whole) {
            float v[RPW][4];
#pragma unroll
            for (int r = 0; r < RPW; ++r) h.x[r].values(v[r]);
            store_rows<VEC, decltype(whole)::value>(out, p, row, nr, v, E4M3);
        });
}

// One CTA per 128 x 128 block, which its threads hold in registers between finding the largest value
// and writing the codes: every element is read once.
constexpr int SQUARE_ROWS = BLOCK / (THREADS / 32);  // rows of a warp
template <typename T, bool VEC, bool E4M3>
__global__ void __launch_bounds__(THREADS) store_square_kernel(const T* x, long ldx, long rows, long cols, Q8 out) {
    __shared__ uint32_t top[THREADS / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long c0 = (long)blockIdx.x * BLOCK + first_col<VEC>(lane);
    const int n = cols - c0 < BLOCK ? (int)(cols - c0) : BLOCK;
    for (long rb = blockIdx.y; rb * BLOCK < rows; rb += gridDim.y) {
        const long r0 = rb * BLOCK + warp * SQUARE_ROWS;
        const int nr = rows - r0 < SQUARE_ROWS ? (int)(rows - r0) : SQUARE_ROWS;
        Raw4<T, VEC> held[SQUARE_ROWS];
        const T* at = x + r0 * ldx + c0;
#pragma unroll
        for (int r = 0; r < SQUARE_ROWS; ++r) held[r].load(at + r * ldx, r < nr ? n : 0);
        uint32_t m = 0, any = 0;
#pragma unroll
        for (int r = 0; r < SQUARE_ROWS; ++r) {
            float v[4];
            held[r].values(v);
            any = max(any, largest(v));
        }
        const bool bad = __syncthreads_or(any > limit_bits(E4M3));
        if (bad) {
#pragma unroll
            for (int r = 0; r < SQUARE_ROWS; ++r) {
                float v[4];
                held[r].values(v);
                limit4(v, E4M3);
                m = max(m, largest_finite(v));
            }
        } else {
            m = any;
        }
        m = __reduce_max_sync(FULL_WARP, m);
        if (lane == 0) top[warp] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < THREADS / 32; ++w) m = max(m, top[w]);
        const uint32_t s = scale_bits(m, E4M3);
        const float inv = inverse_pow2(s);
        uint8_t* q = out.q + r0 * out.ldq + c0;
        if (bad) {
#pragma unroll
            for (int r = 0; r < SQUARE_ROWS; ++r) {
                float v[4];
                held[r].values(v);
                limit4(v, E4M3);
                store_codes<VEC>(q + r * out.ldq, r < nr ? n : 0, encode4(v, inv, E4M3, true));
            }
        } else {
#pragma unroll
            for (int r = 0; r < SQUARE_ROWS; ++r) {
                float v[4];
                held[r].values(v);
                store_codes<VEC>(q + r * out.ldq, r < nr ? n : 0, encode4(v, inv, E4M3, false));
            }
        }
        if (threadIdx.x == 0) out.scale[(long)blockIdx.x * out.lds + rb] = __uint_as_float(s);
        __syncthreads();  // top is read before the next block's is written
    }
}

template <bool VEC>
struct HeldCodes {
    uint32_t w[RPW];
    float s[RPW];
    // shift: log2 of the block's rows
    template <bool WHOLE>
    __device__ __forceinline__ void load(const Q8& t, const Place& p, long row, int nr, int shift) {
        const uint8_t* q = t.q + row * t.ldq + p.col;
        const float* scale = t.scale + (long)p.chunk * t.lds;
#pragma unroll
        for (int r = 0; r < RPW; ++r) {
            w[r] = load_codes<VEC>(q + r * t.ldq, WHOLE || r < nr ? p.n : 0);
            s[r] = WHOLE || r < nr ? scale[(row + r) >> shift] : 0.f;
        }
    }
};

template <typename T, bool VEC, bool E4M3>
__global__ void __launch_bounds__(THREADS) load_kernel(Q8 in, long rows, long cols, int shift, T* y, long ldy) {
    typedef HeldCodes<VEC> Held;
    each_group<VEC, Held>(
        rows, cols,
        [&](const Place& p, Held& h, long row, int nr, auto whole) {
            h.template load<decltype(whole)::value>(in, p, row, nr, shift);
        },
        [&](const Place& p, const Held& h, long row, int nr, auto whole) {
            constexpr bool WHOLE = decltype(whole)::value;
            T* at = y + row * ldy + p.col;
#pragma unroll
            for (int r = 0; r < RPW; ++r) {
                float v[4];
                decode4(h.w[r], E4M3, v);
                uint64_t o[2];
                pairs(v, o);
                o[0] = mul2(o[0], pair(h.s[r]));
                o[1] = mul2(o[1], pair(h.s[r]));
                unpairs(o, v);
                store4<T, VEC>(at + r * ldy, WHOLE || r < nr ? p.n : 0, v);
            }
        });
}

template <typename T, bool VEC, bool E4M3>
__global__ void __launch_bounds__(THREADS)
    gelu_fwd_kernel(const T* z, long ldz, long rows, long cols, T* g, long ldg, Q8 g8, Q8 z8) {
    typedef HeldRows<T, VEC> Held;
    each_group<VEC, Held>(
        rows, cols,
        [&](const Place& p, Held& h, long row, int nr, auto whole) {
            h.template load<decltype(whole)::value>(z + row * ldz + p.col, ldz, p.n, nr);
        },
        [&](const Place& p, const Held& h, long row, int nr, auto whole) {
            constexpr bool WHOLE = decltype(whole)::value;
            float v[RPW][4];
#pragma unroll
            for (int r = 0; r < RPW; ++r) h.x[r].values(v[r]);
            store_rows<VEC, WHOLE>(z8, p, row, nr, v, E4M3);
#pragma unroll
            for (int r = 0; r < RPW; ++r) {
                const uint64_t o[2] = {gelu2(v[r][0], v[r][1]), gelu2(v[r][2], v[r][3])};
                unpairs(o, v[r]);
            }
            if (g) {
                T* to = g + row * ldg + p.col;
#pragma unroll
                for (int r = 0; r < RPW; ++r) store4<T, VEC>(to + r * ldg, WHOLE || r < nr ? p.n : 0, v[r]);
            }
            if (g8.q) store_rows<VEC, WHOLE>(g8, p, row, nr, v, g8.e4m3);
        });
}

template <typename T, bool VEC>
struct HeldBoth {
    HeldRows<T, VEC> x;
    HeldCodes<VEC> c;
};

template <typename T, bool VEC, bool E4M3>
__global__ void __launch_bounds__(THREADS)
    gelu_bwd_kernel(const T* dg, long lddg, Q8 z8, long rows, long cols, T* dz, long lddz, Q8 dz8) {
    typedef HeldBoth<T, VEC> Held;
    each_group<VEC, Held>(
        rows, cols,
        [&](const Place& p, Held& h, long row, int nr, auto whole) {
            constexpr bool WHOLE = decltype(whole)::value;
            h.x.template load<WHOLE>(dg + row * lddg + p.col, lddg, p.n, nr);
            h.c.template load<WHOLE>(z8, p, row, nr, 0);
        },
        [&](const Place& p, const Held& h, long row, int nr, auto whole) {
            constexpr bool WHOLE = decltype(whole)::value;
            float v[RPW][4];
#pragma unroll
            for (int r = 0; r < RPW; ++r) {
                float k[4];
                h.x.x[r].values(v[r]);
                decode4(h.c.w[r], E4M3, k);
                uint64_t k2[2], o[2];
                pairs(k, k2);
                pairs(v[r], o);
#pragma unroll
                for (int i = 0; i < 2; ++i) o[i] = mul2(o[i], gelu_grad2(mul2(k2[i], pair(h.c.s[r]))));
                unpairs(o, v[r]);
            }
            if (dz) {
                T* to = dz + row * lddz + p.col;
#pragma unroll
                for (int r = 0; r < RPW; ++r) store4<T, VEC>(to + r * lddz, WHOLE || r < nr ? p.n : 0, v[r]);
            }
            if (dz8.q) store_rows<VEC, WHOLE>(dz8, p, row, nr, v, dz8.e4m3);
        });
}

// enough warps to fill the GPU (eight CTAs of 256 an SM) or, if there is less, one row group each;
// at least one warp per block column
int grid_for(long rows, long cols) {
    const long chunks = (cols + BLOCK - 1) / BLOCK, groups = (rows + RPW - 1) / RPW;
    const long per = THREADS / 32, full = (long)current_sm_count() * 8 * per;
    long warps = chunks * groups;
    if (warps > full) warps = full > chunks ? full : chunks;
    return (int)((warps + per - 1) / per);
}

template <typename T>
T* as(const OpTensor& t) {
    return static_cast<T*>(const_cast<void*>(t.p));
}

// f(T{}) with T the element type
template <typename Fn>
void by_type(int type, Fn&& f) {
    if (type == OP_F16) f(f16{});
    else if (type == OP_BF16) f(__nv_bfloat16{});
    else f(float{});
}

}  // namespace

void ckpt8_store(const OpTensor& x, long rows, long cols, int block_rows, const Q8& out, cudaStream_t s) {
    const bool v = cols % 4 == 0 && vec4(x) && vec4(out);
    by_type(x.type, [&](auto t) {
        typedef decltype(t) T;
        if (block_rows == 1) {
            auto* k = v ? (out.e4m3 ? store_kernel<T, true, true> : store_kernel<T, true, false>)
                        : (out.e4m3 ? store_kernel<T, false, true> : store_kernel<T, false, false>);
            k<<<grid_for(rows, cols), THREADS, 0, s>>>(as<const T>(x), x.ld, rows, cols, out);
        } else {
            auto* k = v ? (out.e4m3 ? store_square_kernel<T, true, true> : store_square_kernel<T, true, false>)
                        : (out.e4m3 ? store_square_kernel<T, false, true> : store_square_kernel<T, false, false>);
            const long rb = (rows + BLOCK - 1) / BLOCK;
            k<<<dim3((unsigned)((cols + BLOCK - 1) / BLOCK), (unsigned)(rb < 65535 ? rb : 65535)), THREADS, 0, s>>>(
                as<const T>(x), x.ld, rows, cols, out);
        }
    });
}

void ckpt8_load(const Q8& in, long rows, long cols, int block_rows, const OpTensor& y, cudaStream_t s) {
    const bool v = cols % 4 == 0 && vec4(y) && vec4(in);
    by_type(y.type, [&](auto t) {
        typedef decltype(t) T;
        auto* k = v ? (in.e4m3 ? load_kernel<T, true, true> : load_kernel<T, true, false>)
                    : (in.e4m3 ? load_kernel<T, false, true> : load_kernel<T, false, false>);
        k<<<grid_for(rows, cols), THREADS, 0, s>>>(in, rows, cols, block_rows == 1 ? 0 : 7, as<T>(y), y.ld);
    });
}

void gelu_ckpt8_fwd(const OpTensor& z, long rows, long cols, const OpTensor& g, const Q8& g8, const Q8& z8,
                    cudaStream_t s) {
    const bool v = cols % 4 == 0 && vec4(z) && vec4(g) && vec4(g8) && vec4(z8);
    by_type(z.type, [&](auto t) {
        typedef decltype(t) T;
        auto* k = v ? (z8.e4m3 ? gelu_fwd_kernel<T, true, true> : gelu_fwd_kernel<T, true, false>)
                    : (z8.e4m3 ? gelu_fwd_kernel<T, false, true> : gelu_fwd_kernel<T, false, false>);
        k<<<grid_for(rows, cols), THREADS, 0, s>>>(as<const T>(z), z.ld, rows, cols, as<T>(g), g.ld, g8, z8);
    });
}

void gelu_ckpt8_bwd(const OpTensor& dg, const Q8& z8, long rows, long cols, const OpTensor& dz, const Q8& dz8,
                    cudaStream_t s) {
    const bool v = cols % 4 == 0 && vec4(dg) && vec4(dz) && vec4(z8) && vec4(dz8);
    by_type(dg.type, [&](auto t) {
        typedef decltype(t) T;
        auto* k = v ? (z8.e4m3 ? gelu_bwd_kernel<T, true, true> : gelu_bwd_kernel<T, true, false>)
                    : (z8.e4m3 ? gelu_bwd_kernel<T, false, true> : gelu_bwd_kernel<T, false, false>);
        k<<<grid_for(rows, cols), THREADS, 0, s>>>(as<const T>(dg), dg.ld, z8, rows, cols, as<T>(dz), dz.ld, dz8);
    });
}

}  // namespace act
