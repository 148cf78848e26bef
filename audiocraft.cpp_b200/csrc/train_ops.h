// train_ops.h -- launch interface of the operators with weight gradients and 8-bit tensors
// (layer norm, 8-bit checkpoints, rank product from a checkpoint, 8-bit GEMM); the C ABI
// (train_ops.cpp) checks every argument before it gets here.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace act {

enum OpType : int { OP_F32 = 0, OP_F16 = 1, OP_BF16 = 2 };
inline int op_bytes(int type) { return type == OP_F32 ? 4 : 2; }

// codes and block-major scales (null q: absent)
struct Q8 {
    uint8_t* q = nullptr;
    long ldq = 0;
    float* scale = nullptr;  // [ceil(cols / 128)][lds]
    long lds = 0;
    bool e4m3 = false;
};

struct OpTensor {
    const void* p = nullptr;
    int type = OP_F32;
    long ld = 0;
};

// whether base and stride allow four elements to move as one word (with columns a multiple of four
// too, a row's elements all move that way)
inline bool vec4(const OpTensor& t) {
    return !t.p || (t.ld % 4 == 0 && reinterpret_cast<uintptr_t>(t.p) % (4 * op_bytes(t.type)) == 0);
}
inline bool vec4(const Q8& t) { return !t.q || (t.ldq % 4 == 0 && reinterpret_cast<uintptr_t>(t.q) % 4 == 0); }
inline bool vec4(const float* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

void ckpt8_store(const OpTensor& x, long rows, long cols, int block_rows, const Q8& out, cudaStream_t s);
void ckpt8_load(const Q8& in, long rows, long cols, int block_rows, const OpTensor& y, cudaStream_t s);
void gelu_ckpt8_fwd(const OpTensor& z, long rows, long cols, const OpTensor& g, const Q8& g8, const Q8& z8,
                    cudaStream_t s);
void gelu_ckpt8_bwd(const OpTensor& dg, const Q8& z8, long rows, long cols, const OpTensor& dz, const Q8& dz8,
                    cudaStream_t s);

constexpr long LN_MAX_DIM = 8192;
struct LnFwd {
    OpTensor x, y;
    long rows = 0;
    int dim = 0;
    const float *w = nullptr, *b = nullptr;
    float eps = 0.f;
    Q8 y8, x8;
    float *mean = nullptr, *rstd = nullptr;
};
void layernorm_train_fwd(const LnFwd& a, cudaStream_t s);
struct LnBwd {
    OpTensor dy, x, add, dx;
    Q8 x8;
    const float *w = nullptr, *mean = nullptr, *rstd = nullptr;
    long rows = 0;
    int dim = 0;
    float *dw = nullptr, *db = nullptr;
    bool accumulate = false;
    float* space = nullptr;
};
void layernorm_train_bwd(const LnBwd& a, cudaStream_t s);
size_t layernorm_train_bwd_space(long rows, long dim);

struct RankCkpt8 {
    OpTensor u;
    Q8 x;
    int nb = 0;
    long rows = 0, cols = 0;
    float alpha = 1.f;
    float* c = nullptr;
    long ldc = 0;
    bool accumulate = false;
    int* status = nullptr;
};
void rank_ckpt8(const RankCkpt8& a, cudaStream_t s);

struct GemmF8 {
    Q8 x, w;
    long M = 0, N = 0, K = 0;
    bool w_mn = false;
    const float* bias = nullptr;
    OpTensor y;
    bool accumulate = false;
    int* status = nullptr;
};
void gemm_f8(const GemmF8& a, cudaStream_t s);

}  // namespace act
