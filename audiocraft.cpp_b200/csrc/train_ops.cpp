// train_ops.cpp -- C ABI of the operators with weight gradients and 8-bit tensors: checks of
// every argument before any work is queued, then one or two launches on the caller's stream.
#include "train_ops.h"

#include <cmath>
#include <stdexcept>
#include <string>

#include "actrain.h"
#include "kernels.h"

namespace {

using act::OpTensor;
using act::Q8;

constexpr int64_t kMaxSize = 1ll << 31;  // rows, columns and strides fit an int

// Thrown by the checks, turned into a status at the C entry
struct Refused : std::runtime_error {
    int code;
    Refused(int c, const std::string& m) : std::runtime_error(m), code(c) {}
};
[[noreturn]] void refuse(const std::string& m) { throw Refused(ACT_ERR_INVALID, m); }

struct Checker {
    std::string name;
    int device = -1;
    explicit Checker(const char* n) : name(n) {}

    void size(int64_t v, int64_t lo, int64_t hi, const char* what) const {
        if (v < lo || v > hi)
            refuse(name + ": " + what + " is " + std::to_string(v) + ", must be " + std::to_string(lo) + " .. " +
                   std::to_string(hi));
    }
    void flag(int v, const char* what) const { size(v, 0, 1, what); }

    // Device memory of the current device?  Asked once the shapes are right; a host pointer or
    // another device's would fault on the GPU.
    void where(const void* p, const char* what) {
        if (device < 0) {
            const cudaError_t e = cudaGetDevice(&device);
            if (e != cudaSuccess) {
                cudaGetLastError();
                throw Refused(ACT_ERR_CUDA, name + ": cudaGetDevice: " + cudaGetErrorString(e));
            }
        }
        cudaPointerAttributes at;
        const cudaError_t e = cudaPointerGetAttributes(&at, p);
        if (e != cudaSuccess) {
            cudaGetLastError();
            throw Refused(ACT_ERR_CUDA, name + ": cudaPointerGetAttributes: " + cudaGetErrorString(e));
        }
        if (at.type == cudaMemoryTypeManaged) return;
        if (at.type != cudaMemoryTypeDevice) refuse(name + ": " + what + " is not device memory");
        if (at.device != device)
            refuse(name + ": " + what + " is on device " + std::to_string(at.device) + ", the current device is " +
                   std::to_string(device));
    }
    // rows: of the tensor; one without any may be NULL, as the address of an empty tensor is
    void raw(const void* p, size_t align, const char* what, int64_t rows = 1) const {
        if (!p && rows == 0) return;
        if (!p) refuse(name + ": " + what + " is NULL");
        if (reinterpret_cast<uintptr_t>(p) % align)
            refuse(name + ": " + what + " must be " + std::to_string(align) + "-byte aligned");
    }
    int type(int ggml, const char* what) const {
        if (ggml == ACT_TYPE_F32) return act::OP_F32;
        if (ggml == ACT_TYPE_F16) return act::OP_F16;
        if (ggml == ACT_TYPE_BF16) return act::OP_BF16;
        refuse(name + ": " + what + " type " + std::to_string(ggml) + " (ACT_TYPE_F32, _F16 or _BF16)");
    }
    OpTensor tensor(const void* p, int ggml, int64_t ld, int64_t rows, int64_t cols, const char* what) const {
        OpTensor t;
        t.type = type(ggml, what);
        raw(p, act::op_bytes(t.type), what, rows);
        if (ld < cols || ld > kMaxSize)
            refuse(name + ": row stride of " + what + " is " + std::to_string(ld) + " for " + std::to_string(cols) +
                   " columns");
        t.p = p;
        t.ld = ld;
        return t;
    }
    // pitch: alignment of the codes' rows
    Q8 codes(const act_ckpt8* v, int64_t rows, int64_t cols, int block_rows, int64_t pitch, const char* what) const {
        if (!v) refuse(name + ": " + what + " is NULL");
        if (v->type != ACT_CKPT_I8 && v->type != ACT_CKPT_E4M3)
            refuse(name + ": " + what + " has type " + std::to_string(v->type) + " (ACT_CKPT_I8 or _E4M3)");
        raw(v->q, pitch, what, rows);
        raw(v->scale, 4, (std::string(what) + "'s scale").c_str(), rows);
        if (v->ldq < cols || v->ldq > kMaxSize || v->ldq % pitch)
            refuse(name + ": row stride of " + what + " is " + std::to_string(v->ldq) + " for " +
                   std::to_string(cols) + " columns (a multiple of " + std::to_string(pitch) + ")");
        const int64_t need = (rows + block_rows - 1) / block_rows;
        if (v->lds < need || v->lds > kMaxSize)
            refuse(name + ": " + what + " has " + std::to_string(v->lds) + " scales a block column, needs " +
                   std::to_string(need));
        Q8 t;
        t.q = static_cast<uint8_t*>(v->q);
        t.ldq = v->ldq;
        t.scale = v->scale;
        t.lds = v->lds;
        t.e4m3 = v->type == ACT_CKPT_E4M3;
        return t;
    }
    void where(const Q8& t, const char* what) {
        if (!t.q) return;
        where(t.q, what);
        where(t.scale, what);
    }
    void where(const OpTensor& t, const char* what) {
        if (t.p) where(t.p, what);
    }
    void done() const {
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) throw Refused(ACT_ERR_CUDA, name + " launch: " + cudaGetErrorString(e));
    }
};

// no C++ exception may cross the C ABI
template <typename Fn>
int guarded(const char* name, Fn&& fn) {
    try {
        Checker c(name);
        fn(c);
        return ACT_OK;
    } catch (const Refused& e) {
        try {
            act::set_last_error(e.what());
        } catch (...) {
        }
        return e.code;
    } catch (const std::exception& e) {
        try {
            act::set_last_error(std::string(name) + ": " + e.what());
        } catch (...) {
        }
        return ACT_ERR_CUDA;
    } catch (...) {
        return ACT_ERR_CUDA;
    }
}

cudaStream_t on(void* s) { return static_cast<cudaStream_t>(s); }

void block(const Checker& c, int block_rows) {
    if (block_rows != 1 && block_rows != 128)
        refuse(c.name + ": block_rows is " + std::to_string(block_rows) + ", must be 1 or 128");
}

}  // namespace

extern "C" int act_ckpt8_store(const void* x, int x_type, int64_t ldx, int64_t rows, int64_t cols, int block_rows,
                               const act_ckpt8* out, void* stream) {
    return guarded("act_ckpt8_store", [&](Checker& c) {
        c.size(rows, 0, kMaxSize - 1, "rows");
        c.size(cols, 1, kMaxSize - 1, "cols");
        block(c, block_rows);
        const OpTensor tx = c.tensor(x, x_type, ldx, rows, cols, "x");
        const Q8 t = c.codes(out, rows, cols, block_rows, 1, "out");
        if (!rows) return;
        c.where(tx, "x");
        c.where(t, "out");
        act::ckpt8_store(tx, rows, cols, block_rows, t, on(stream));
        c.done();
    });
}

extern "C" int act_ckpt8_load(const act_ckpt8* in, int64_t rows, int64_t cols, int block_rows, void* y, int y_type,
                              int64_t ldy, void* stream) {
    return guarded("act_ckpt8_load", [&](Checker& c) {
        c.size(rows, 0, kMaxSize - 1, "rows");
        c.size(cols, 1, kMaxSize - 1, "cols");
        block(c, block_rows);
        const OpTensor ty = c.tensor(y, y_type, ldy, rows, cols, "y");
        const Q8 t = c.codes(in, rows, cols, block_rows, 1, "in");
        if (!rows) return;
        c.where(t, "in");
        c.where(ty, "y");
        act::ckpt8_load(t, rows, cols, block_rows, ty, on(stream));
        c.done();
    });
}

extern "C" int act_layernorm_fwd(const void* x, int x_type, int64_t ldx, int64_t rows, int64_t dim, const float* w,
                                 const float* b, float eps, void* y, int y_type, int64_t ldy, const act_ckpt8* y8,
                                 float* mean, float* rstd, const act_ckpt8* x8, void* stream) {
    return guarded("act_layernorm_fwd", [&](Checker& c) {
        c.size(rows, 0, kMaxSize - 1, "rows");
        c.size(dim, 1, act::LN_MAX_DIM, "dim");
        if (!(eps >= 0.f) || std::isinf(eps)) refuse(c.name + ": eps must be finite and not negative");
        if (rows && !y && !y8) refuse(c.name + ": y and y8 are both NULL");
        act::LnFwd a;
        a.x = c.tensor(x, x_type, ldx, rows, dim, "x");
        if (y) a.y = c.tensor(y, y_type, ldy, rows, dim, "y");
        if (y8) a.y8 = c.codes(y8, rows, dim, 1, 1, "y8");
        if (x8) a.x8 = c.codes(x8, rows, dim, 1, 1, "x8");
        if (w) c.raw(w, 4, "w");
        if (b) c.raw(b, 4, "b");
        c.raw(mean, 4, "mean", rows);
        c.raw(rstd, 4, "rstd", rows);
        if (!rows) return;
        c.where(a.x, "x");
        c.where(a.y, "y");
        c.where(a.y8, "y8");
        c.where(a.x8, "x8");
        if (w) c.where(w, "w");
        if (b) c.where(b, "b");
        c.where(mean, "mean");
        c.where(rstd, "rstd");
        a.rows = rows; a.dim = (int)dim; a.w = w; a.b = b; a.eps = eps; a.mean = mean; a.rstd = rstd;
        act::layernorm_train_fwd(a, on(stream));
        c.done();
    });
}

extern "C" int64_t act_layernorm_bwd_workspace(int64_t rows, int64_t dim) {
    int64_t bytes = -1;
    guarded("act_layernorm_bwd_workspace", [&](Checker& c) {
        c.size(rows, 0, kMaxSize - 1, "rows");
        c.size(dim, 1, act::LN_MAX_DIM, "dim");
        bytes = (int64_t)act::layernorm_train_bwd_space(rows, dim);
    });
    return bytes;
}

extern "C" int act_layernorm_bwd(const void* dy, int dy_type, int64_t lddy, const void* x, int x_type, int64_t ldx,
                                 const act_ckpt8* x8, const float* w, const float* mean, const float* rstd,
                                 int64_t rows, int64_t dim, const void* add, void* dx, int dx_type, int64_t lddx,
                                 float* dw, float* db, int accumulate, void* workspace, size_t workspace_bytes,
                                 void* stream) {
    return guarded("act_layernorm_bwd", [&](Checker& c) {
        c.size(rows, 0, kMaxSize - 1, "rows");
        c.size(dim, 1, act::LN_MAX_DIM, "dim");
        c.flag(accumulate, "accumulate");
        if (x ? x8 != nullptr : !x8 && rows) refuse(c.name + ": exactly one of x and x8 must be given");
        act::LnBwd a;
        a.dy = c.tensor(dy, dy_type, lddy, rows, dim, "dy");
        if (x) a.x = c.tensor(x, x_type, ldx, rows, dim, "x");
        if (x8) a.x8 = c.codes(x8, rows, dim, 1, 1, "x8");
        a.dx = c.tensor(dx, dx_type, lddx, rows, dim, "dx");
        if (add) a.add = c.tensor(add, dx_type, lddx, rows, dim, "add");
        if (w) c.raw(w, 4, "w");
        c.raw(mean, 4, "mean", rows);
        c.raw(rstd, 4, "rstd", rows);
        if (dw) c.raw(dw, 4, "dw");
        if (db) c.raw(db, 4, "db");
        c.raw(workspace, 16, "workspace");
        const size_t need = act::layernorm_train_bwd_space(rows, dim);
        if (workspace_bytes < need)
            refuse(c.name + ": workspace holds " + std::to_string(workspace_bytes) + " bytes, needs " +
                   std::to_string(need));
        if (rows || ((dw || db) && !accumulate)) {
            c.where(workspace, "workspace");
            if (dw) c.where(dw, "dw");
            if (db) c.where(db, "db");
        }
        if (rows) {
            c.where(a.dy, "dy");
            c.where(a.x, "x");
            c.where(a.x8, "x8");
            c.where(a.add, "add");
            c.where(a.dx, "dx");
            if (w) c.where(w, "w");
            c.where(mean, "mean");
            c.where(rstd, "rstd");
        } else if (accumulate || (!dw && !db)) {
            return;
        }
        a.w = w; a.mean = mean; a.rstd = rstd; a.rows = rows; a.dim = (int)dim; a.dw = dw; a.db = db;
        a.accumulate = accumulate != 0;
        a.space = static_cast<float*>(workspace);
        act::layernorm_train_bwd(a, on(stream));
        c.done();
    });
}

extern "C" int act_gelu_ckpt8_fwd(const void* z, int z_type, int64_t ldz, int64_t rows, int64_t cols, void* g,
                                  int64_t ldg, const act_ckpt8* g8, const act_ckpt8* z8, void* stream) {
    return guarded("act_gelu_ckpt8_fwd", [&](Checker& c) {
        c.size(rows, 0, kMaxSize - 1, "rows");
        c.size(cols, 1, kMaxSize - 1, "cols");
        if (rows && !g && !g8) refuse(c.name + ": g and g8 are both NULL");
        const OpTensor tz = c.tensor(z, z_type, ldz, rows, cols, "z");
        OpTensor tg;
        Q8 t8;
        if (g) tg = c.tensor(g, z_type, ldg, rows, cols, "g");
        if (g8) t8 = c.codes(g8, rows, cols, 1, 1, "g8");
        const Q8 tk = c.codes(z8, rows, cols, 1, 1, "z8");
        if (!rows) return;
        c.where(tz, "z");
        c.where(tg, "g");
        c.where(t8, "g8");
        c.where(tk, "z8");
        act::gelu_ckpt8_fwd(tz, rows, cols, tg, t8, tk, on(stream));
        c.done();
    });
}

extern "C" int act_gelu_ckpt8_bwd(const void* dg, int dg_type, int64_t lddg, const act_ckpt8* z8, int64_t rows,
                                  int64_t cols, void* dz, int64_t lddz, const act_ckpt8* dz8, void* stream) {
    return guarded("act_gelu_ckpt8_bwd", [&](Checker& c) {
        c.size(rows, 0, kMaxSize - 1, "rows");
        c.size(cols, 1, kMaxSize - 1, "cols");
        if (rows && !dz && !dz8) refuse(c.name + ": dz and dz8 are both NULL");
        const OpTensor tg = c.tensor(dg, dg_type, lddg, rows, cols, "dg");
        const Q8 tk = c.codes(z8, rows, cols, 1, 1, "z8");
        OpTensor tz;
        Q8 t8;
        if (dz) tz = c.tensor(dz, dg_type, lddz, rows, cols, "dz");
        if (dz8) t8 = c.codes(dz8, rows, cols, 1, 1, "dz8");
        if (!rows) return;
        c.where(tg, "dg");
        c.where(tk, "z8");
        c.where(tz, "dz");
        c.where(t8, "dz8");
        act::gelu_ckpt8_bwd(tg, tk, rows, cols, tz, t8, on(stream));
        c.done();
    });
}

extern "C" int act_rank_gemm_ckpt8(const void* u, int u_type, int64_t ldu, int nb, const act_ckpt8* x, int64_t rows,
                                   int64_t cols, float alpha, float* cp, int64_t ldc, int accumulate,
                                   int32_t* status, void* stream) {
    return guarded("act_rank_gemm_ckpt8", [&](Checker& c) {
        c.size(rows, 0, kMaxSize - 1, "rows");
        c.size(cols, 1, kMaxSize - 1, "cols");
        c.size(nb, 1, 64, "nb");
        c.flag(accumulate, "accumulate");
        act::RankCkpt8 a;
        a.u = c.tensor(u, u_type, ldu, rows, nb, "u");
        a.x = c.codes(x, rows, cols, 1, 16, "x");
        c.tensor(cp, ACT_TYPE_F32, ldc, nb, cols, "c");
        c.raw(status, 4, "status");
        if (!rows && accumulate) return;
        if (rows) {
            c.where(a.u, "u");
            c.where(a.x, "x");
        }
        c.where(cp, "c");
        c.where(status, "status");
        a.nb = nb; a.rows = rows; a.cols = cols; a.alpha = alpha; a.c = cp; a.ldc = ldc;
        a.accumulate = accumulate != 0;
        a.status = status;
        act::rank_ckpt8(a, on(stream));
        c.done();
    });
}

extern "C" int act_copy_wait_probe(const void* src, void* dst, int64_t limit_ns, int32_t* status, void* stream) {
    return guarded("act_copy_wait_probe", [&](Checker& c) {
        c.size(limit_ns, 1, 10000000000ll, "limit_ns");
        c.raw(src, 16, "src");
        c.raw(dst, 1, "dst");
        c.raw(status, 4, "status");
        c.where(src, "src");
        c.where(dst, "dst");
        c.where(status, "status");
        act::copy_wait_probe(src, dst, limit_ns, status, on(stream));
        c.done();
    });
}

extern "C" int act_gemm_f8(const act_ckpt8* x, const act_ckpt8* w, int64_t M, int64_t N, int64_t K, int w_mn_major,
                           const float* bias, void* y, int y_type, int64_t ldy, int accumulate, int32_t* status,
                           void* stream) {
    return guarded("act_gemm_f8", [&](Checker& c) {
        c.size(M, 0, kMaxSize - 1, "M");
        c.size(N, 1, kMaxSize - 1, "N");
        c.size(K, 1, kMaxSize - 1, "K");
        c.flag(w_mn_major, "w_mn_major");
        c.flag(accumulate, "accumulate");
        act::GemmF8 a;
        a.x = c.codes(x, M, K, 1, 16, "x");
        a.w = w_mn_major ? c.codes(w, K, N, 128, 16, "w") : c.codes(w, N, K, 128, 16, "w");
        if (!a.x.e4m3 || !a.w.e4m3) refuse(c.name + ": x and w must be ACT_CKPT_E4M3");
        if (bias) c.raw(bias, 4, "bias");
        a.y = c.tensor(y, y_type, ldy, M, N, "y");
        c.raw(status, 4, "status");
        if (!M) return;
        c.where(a.x, "x");
        c.where(a.w, "w");
        if (bias) c.where(bias, "bias");
        c.where(a.y, "y");
        c.where(status, "status");
        a.M = M; a.N = N; a.K = K; a.w_mn = w_mn_major != 0; a.bias = bias; a.accumulate = accumulate != 0;
        a.status = status;
        act::gemm_f8(a, on(stream));
        c.done();
    });
}
