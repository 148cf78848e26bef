/*
 * actrain.h -- C ABI of the B200 adapter-training step (libactrain.so).
 *
 * This is the seam between the unchanged trainer front ends (mf-train / mg-train argument
 * parsing, cache sampling, checkpoint files) and the device step.  In the reference the
 * same seam is the class API of MfTrainGraph / MgTrainGraph plus TrainAccumulation:
 *   src/mf/train.h:31-256      MfTrainGraph  (ctor, compute, compute_bridge, adam_step, save)
 *   src/mg/train.h:51-230      MgTrainGraph  (ctor, compute, adam_step, save)
 *   src/ac/train_controls.h:75-119  TrainAccumulation (add, update)
 *   src/gguf_model.h:363-436   load_gguf / graph_compute_checked (weights on the device)
 *
 * Conventions: every call returns ACT_OK (0) or a nonzero status and never throws; the
 * message of the last failure is available from act_last_error().  A context is bound to
 * one CUDA device and is not thread-safe: one host thread per rank.  All pointers in the
 * batch structs are HOST pointers unless a name says otherwise.
 */
#ifndef ACTRAIN_H
#define ACTRAIN_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif
#if defined(__GNUC__)
#pragma GCC visibility push(default)
#endif

#define ACT_OK 0
#define ACT_ERR_INVALID 1    /* bad argument, shape or configuration (reference: std::runtime_error) */
#define ACT_ERR_CUDA 2       /* CUDA runtime failure */
#define ACT_ERR_NCCL 3       /* NCCL failure */
#define ACT_ERR_STATE 4      /* call out of order (e.g. step before act_finalize) */
#define ACT_ERR_NONFINITE 5  /* nonfinite loss or optimizer update (src/mf/train.h:186, train_controls.h:113) */

#define ACT_FAMILY_MELODYFLOW 0
#define ACT_FAMILY_MUSICGEN 1

#define ACT_ADAPTER_LORA 0
#define ACT_ADAPTER_DORA_ROWS 1

/* ggml type ids of the base weights accepted by act_bind_weight */
#define ACT_TYPE_F32 0
#define ACT_TYPE_F16 1
#define ACT_TYPE_Q8_0 8
#define ACT_TYPE_BF16 30 /* the 8-bit checkpoint, layer norm and 8-bit GEMM entry points below only */

/* adapter target bits, in the reference's order (src/mf/train.h:69, src/mg/train.h:90) */
#define ACT_TARGET_SELF_QKV (1u << 0)
#define ACT_TARGET_SELF_OUT (1u << 1)
#define ACT_TARGET_CROSS_Q (1u << 2)
#define ACT_TARGET_CROSS_KV (1u << 3)
#define ACT_TARGET_CROSS_OUT (1u << 4)
#define ACT_TARGET_FF0 (1u << 5)
#define ACT_TARGET_FF2 (1u << 6)
#define ACT_TARGETS_REFERENCE 0x1Fu     /* attention projections (default mf-train / mg-train) */
#define ACT_TARGETS_REFERENCE_FFN 0x7Fu /* with --train-ffn */

typedef struct act_ctx act_ctx;

/* Model hyper-parameters, read by the caller from GGUF metadata exactly as
 * DitConfig::from (src/mf/dit.h:44-71) and LmConfig::from (src/mg/lm.h:60-90) do. */
typedef struct {
    int family;                                  /* ACT_FAMILY_* */
    int dim, layers, heads, head_dim, ff_dim;
    int latent_dim, cond_dim, time_dim, n_skip;  /* MelodyFlow */
    int add_zero_attn;                           /* MelodyFlow */
    int n_q, card, special_token_id, pos_denominator; /* MusicGen */
    float max_period;                            /* MusicGen sin positions */
    float norm_eps;
} act_model_desc;

/* Adapter and capacity: MfTrainGraph(W, c, frames, tokens, rank, alpha, first_layer, seed,
 * type, feedforward) (src/mf/train.h:47-48) / MgTrainGraph(..., prefix, ...) (src/mg/train.h:66-67).
 * `targets` generalises the reference's feedforward flag (0x1F / 0x7F reproduce it). */
typedef struct {
    int type;          /* ACT_ADAPTER_LORA | ACT_ADAPTER_DORA_ROWS */
    int rank;
    float alpha;       /* scale = alpha / rank */
    int first_layer;
    unsigned targets;  /* ACT_TARGET_* bits */
    uint32_t seed;     /* lora_A ~ N(0, 0.02) drawn from std::mt19937(seed) in parameter order */
    int max_batch;     /* clips (MelodyFlow) or sequences (MusicGen) per step on this device */
    int frames;        /* latent frames (MelodyFlow) / codec timesteps (MusicGen) */
    int tokens;        /* conditioning tokens */
    int prefix_frames; /* MusicGen: timesteps before this are not scored (src/mg/train.h:195-196) */
} act_adapter_desc;

/* One MelodyFlow microbatch (MfTrainGraph::compute, src/mf/train.h:148-188), n <= max_batch. */
typedef struct {
    int n;
    const float* clean;        /* [n][latent_dim][frames] */
    const float* noise;        /* [n][latent_dim][frames] */
    const float* hidden;       /* [n][tokens][cond_dim] T5 states (zero padded) */
    const float* t;            /* [n] flow time in [0, 1] */
    const int32_t* unconditional; /* [n] or NULL: 1 masks every text token */
    const int32_t* valid_tokens;  /* [n] or NULL: tokens >= valid are masked; -1 = all */
    /* Edit-bridge objective (MfTrainGraph::compute_bridge, src/mf/train.h:190-204), or NULL for
     * flow matching.  The straight bridge x_t = (1-u) pivot + u clean, u = (t-start)/(1-start),
     * is trained through its equivalent t = 0 endpoint (pivot - start*clean) / (1 - start), which
     * the device forms in place of noise (noise may then be NULL).  Needs 0 <= start < 1 and
     * start <= t <= 1 for every sample. */
    const float* pivot;           /* [n][latent_dim][frames] */
    const float* edit_start;      /* [n] */
    /* On-device sampling (the reference draws these on the host, tools/mf-train.cpp:250-262):
     * when stddev is given, `clean` holds the posterior mean and the device draws clean = mean +
     * stddev * z and noise = z' (z, z' ~ N(0,1), Box-Muller from Philox4x32-10 keyed by
     * sample_seed, counted by window number window0 + i and element), and `noise` is ignored.
     * Reproducible per (seed, window, element), not the reference's host random stream.  Not
     * with pivot. */
    const float* stddev;          /* [n][latent_dim][frames] or NULL */
    uint64_t sample_seed;
    uint64_t window0;
} act_mf_batch;

/* One MusicGen microbatch (MgTrainGraph::compute, src/mg/train.h:178-227). */
typedef struct {
    int n;
    const int32_t* codes;      /* [n][n_q][frames] codec tokens in [0, card) */
    const float* context;      /* [n][tokens][dim] projected conditioning */
} act_mg_batch;

/* TrainAccumulation::update (src/ac/train_controls.h:89-118). */
typedef struct {
    float lr;            /* already scheduled: TrainControls::rate (src/ac/train_controls.h:53-58) */
    float beta1, beta2, eps;
    float weight_decay;  /* decoupled; applied to lora_A / lora_B only */
    float clip;          /* global L2 clip */
    int step;            /* 1-based optimizer step for bias correction */
    int count;           /* samples the gradient sum averages over; 0 = accumulated count */
} act_opt;

/* replaces the MfTrainGraph / MgTrainGraph constructors (graph build + allocation) */
int act_create(act_ctx** out, int device, const act_model_desc* model, const act_adapter_desc* adapter);
/* replaces load_gguf's tensor upload (src/gguf_model.h:363-420); name = GGUF tensor name */
int act_bind_weight(act_ctx* ctx, const char* name, int ggml_type, const void* host, size_t bytes);
/* after every weight: checks completeness, DoRA row norms (src/ac/lora.h:11-32), parameter init */
int act_finalize(act_ctx* ctx);

/* parameter table in the reference order (src/mf/train.h:68-104): name, flat offset, shape */
int64_t act_param_count(act_ctx* ctx);
int act_param_tensor_count(act_ctx* ctx);
int act_param_tensor(act_ctx* ctx, int index, char* name, size_t name_cap, int64_t* offset,
                     int64_t* rows, int64_t* cols);
int act_set_params(act_ctx* ctx, const float* value, size_t n);
/* value, m, v (any may be NULL): what save() and the .state sidecar write */
int act_get_params(act_ctx* ctx, float* value, float* m, float* v, size_t n);
int act_set_moments(act_ctx* ctx, const float* m, const float* v, size_t n);
int act_get_grads(act_ctx* ctx, float* grad, size_t n);
int act_zero_grads(act_ctx* ctx);

/* forward + backward of one microbatch; gradients accumulate on the device (the reference's
 * compute() followed by TrainAccumulation::add).  loss_per_sample may be NULL. */
int act_mf_step(act_ctx* ctx, const act_mf_batch* batch, float* loss_per_sample);
int act_mg_step(act_ctx* ctx, const act_mg_batch* batch, float* loss_per_sample);

/* data parallelism (no counterpart in the reference, which trains on one device) */
int act_nccl_get_unique_id(void* id_128_bytes);
int act_nccl_init(act_ctx* ctx, const void* id_128_bytes, int nranks, int rank);
/* sum gradients over ranks; nccl_comm NULL uses the context's own communicator.
 * global_count becomes the averaging count of the next act_optimizer. */
int act_allreduce_grads(act_ctx* ctx, void* nccl_comm, int global_count);
/* The next step (act_mf_step / act_mg_step / act_run_staged) all-reduces the gradients inside
 * the step, over the context's communicator: each layer's gradients start their all-reduce as
 * soon as that layer's backward has been issued (DoRA: once, after the whole backward), on a
 * stream of their own that overlaps the remaining backward.  It takes the place of
 * act_allreduce_grads after the last microbatch of an accumulation; global_count becomes the
 * averaging count of the next act_optimizer.  0 cancels. */
int act_set_grad_sync(act_ctx* ctx, int global_count);
/* Bit-for-bit reproducible steps (1) or the default (0).  Every reduction of the step is
 * order-independent except the self-attention backward's dQ, whose key blocks add their tiles
 * into one fp32 accumulator as they finish; with 1 they add in key-block order (each waits for
 * its predecessors, bounded), which makes the whole step a pure function of its inputs at the
 * cost of about 1.5 ms per cfg-2 step (5%).  The trainer front ends turn it on: exact resume and
 * checkpoints that leave training unchanged depend on it. */
int act_set_deterministic(act_ctx* ctx, int enable);
/* Bound, in milliseconds, on NCCL initialisation and on every host wait for the device while
 * a communicator is live (0 = none, the default).  A rank that stalls or dies makes the others'
 * next wait expire: their communicator is aborted (ncclCommAbort) and the call returns
 * ACT_ERR_NCCL instead of blocking forever. */
int act_set_timeout(act_ctx* ctx, int64_t timeout_ms);

/* mean, clip, AdamW, zero gradients (TrainAccumulation::update).  *nonfinite receives the
 * number of nonfinite updated values; a nonzero count also returns ACT_ERR_NONFINITE. */
int act_optimizer(act_ctx* ctx, const act_opt* opt, int* nonfinite);

const char* act_last_error(act_ctx* ctx);
void act_destroy(act_ctx* ctx);

/* ---- measurement hooks (device-resident inputs, kernel timing) ---- */
void* act_stream(act_ctx* ctx);   /* the cudaStream_t every kernel of the context runs on */
/* copy a batch to the device (host->device), then run it from device memory */
int act_mf_stage(act_ctx* ctx, const act_mf_batch* batch);
int act_mg_stage(act_ctx* ctx, const act_mg_batch* batch);
int act_run_staged(act_ctx* ctx, float* loss_per_sample /* may be NULL: no device->host read */);
/* per-kernel-class timing of eagerly launched steps: 0 disables (steps use the CUDA graph) */
int act_set_profiling(act_ctx* ctx, int enable);
/* class 0 = dense projection GEMMs, 1 = attention fwd+bwd, 2 = everything else */
int act_kernel_stats(act_ctx* ctx, int cls, double* ms, double* flops, double* bytes, int64_t* launches);
int act_reset_kernel_stats(act_ctx* ctx);
/* algorithmic FLOPs of one step of n samples (2 per multiply-add) */
double act_step_flops(act_ctx* ctx, int n);
/* stand-alone projection GEMM on host buffers (tests and the kernel sweep): C[M][N] fp32 =
 * A[M][K] . B(n,k) with f16 A and B, B as [N][K] (b_mn_major 0) or [K][N] (1);
 * path 0 = automatic, 1 = mma.sync kernel, 2 = tcgen05 kernel, 3 = tcgen05 2-CTA (cta_group::2)
 * kernel (stream-K split of the tiles where whole tiles would leave the last round mostly
 * idle), 4 = the 2-CTA kernel with 128-column pair tiles, 5 = the 2-CTA kernel on whole
 * tiles only; when reps > 0 the GEMM is
 * re-run reps times back to back and *ms_per_call receives the mean device time */
int act_gemm_f16(int device, const void* A, const void* B, void* C, int M, int N, int K, int b_mn_major, int path,
                 int reps, float* ms_per_call);
/* The same with B given as the Q8_0 blocks (34 bytes each, tools/ac-quantize.cpp:161) of the
 * weight [N][K] (b_mn_major 0) or [K][N] (1), kept quantised on the device: the 2-CTA kernel's
 * converter warps dequantise each k-block in shared memory (paths 0, 3, 4, 5).  The MMA sees the
 * values act_q8_0_dequant gives, so C equals act_gemm_f16 on that dequantised B bit for bit when
 * both run the same tile schedule (paths 4 and 5). */
int act_gemm_q8_0(int device, const void* A, const void* Bq8, void* C, int M, int N, int K, int b_mn_major, int path,
                  int reps, float* ms_per_call);
/* stand-alone rank-block product (tests and the kernel sweep): C = alpha * A(M x K) B(K x nb),
 * nb <= 64, f16 A stored [M][K] (a_mn 0) or [K][M] (1), f16 B stored [nb][K] (b_mn 0) or
 * [K][nb] (1).  kind 0: C [M][nb] fp32 += result; kind 1: C [nb][M] fp32 += result transposed;
 * kind 2: C [M][nb] = the result rounded to f16 (returned as fp32).  splits 0 = automatic.
 * No reference counterpart: the reference evaluates these products as separate ggml mul_mat
 * nodes (src/ac/lora.h:34-95).  When reps > 0 the call is re-run reps times (kind 0/1 keep
 * accumulating) and *ms_per_call receives the mean device time. */
/* stand-alone check of the feed-forward activation: g = f16(gelu(z)), dg = f16(gelu'(z)) for
 * f16 z (A&S 7.1.26 GELU of src/ac/lora.h:97-110 and the derivative of that approximation),
 * evaluated element by element (direct = 1) or by the vectorised pass the training step runs,
 * which overwrites the pre-activation with gelu' (0); the two agree bit for bit. */
int act_gelu_f16(int device, const uint16_t* z, uint16_t* g, uint16_t* dg, int64_t n, int direct);
int act_rank_gemm_f16(int device, int kind, const void* A, const void* B, float* C, int M, int K, int nb, int a_mn,
                      int b_mn, float alpha, int splits, int reps, float* ms_per_call);
/* The same product with A read from a frozen weight given as its Q8_0 blocks (34 bytes each,
 * tools/ac-quantize.cpp:161): the weight is [M][K] (a_mn 0) or [K][M] (1) and stays quantised on
 * the device; the kernel's converter warps dequantise each k-block on its way into the MMA (the
 * DoRA products P = W A^T and BD^T W of the training step, src/ac/lora.h:62-79).  With the same
 * splits, C equals act_rank_gemm_f16 on the act_q8_0_dequant f16 values bit for bit. */
int act_rank_gemm_q8_0(int device, int kind, const void* Aq8, const void* B, float* C, int M, int K, int nb, int a_mn,
                       int b_mn, float alpha, int splits, int reps, float* ms_per_call);
/* stand-alone attention forward + backward on host buffers (tests and the kernel sweep):
 * token-major f16 q [clips*T][H*64], k/v [clips*Tk][H*64], dout like q; scale 1/8 (head_dim 64);
 * nvalid: per-clip valid key count or NULL; causal; zero_key = the prepended zero key of
 * src/ac/transformer.h:74-79; rope: [T][32] (cos, sin) pairs or NULL.  Outputs o (f16),
 * lse (fp32 [clips][H][T], base-2 log-sum-exp of the scaled scores), and, when dout is given,
 * dq (f16, like q), dk / dv (f16, like k).  ms_fwd / ms_bwd (nullable) receive device times. */
int act_attention(int device, const void* q, const void* k, const void* v, const void* dout, int clips, int T,
                  int Tk, int H, const int32_t* nvalid, int causal, int zero_key, const float* rope, void* o,
                  float* lse, void* dq, void* dk, void* dv, float* ms_fwd, float* ms_bwd);
/* ---- attention backward that allocates nothing (no counterpart in the reference) ----
 * For callers that must not call cudaMalloc / cudaFree: real-time hosts such as an audio
 * plug-in's processing thread (an allocation can block and synchronise the device), code
 * recording a CUDA graph under global stream capture (allocation is not permitted there), and
 * embedders that own all device memory through their own pool.  Same computation and layouts
 * as the backward half of act_attention, but every pointer is a DEVICE pointer on the calling
 * thread's current device (nvalid and rope too), o and lse come from a forward pass, and the
 * work is queued asynchronously on `stream` (NULL = the legacy default stream).
 * Scratch (the fp32 dQ accumulator and the per-row rowsum(dO*O)) lives in one fixed array of
 * ACT_NOALLOC_ATTN_SCRATCH_FLOATS floats (32 MiB) compiled into the library; every GPU that
 * loads the library holds it until the process exits.  A problem needing more than
 * clips*T*H*64 + clips*H*T <= ACT_NOALLOC_ATTN_SCRATCH_FLOATS floats is rejected with
 * ACT_ERR_INVALID.  The first call on each device looks up that device's copy of the array
 * (cudaGetSymbolAddress); make that first call before any stream capture, and do not reset the
 * device (cudaDeviceReset or a primary-context reset) afterwards: the looked-up address is kept
 * for the life of the process.  Every call uses the same array and zeroes the accumulator it
 * needs, so calls that overlap on the GPU (on different streams, or from different threads)
 * race: serialise them.  q, k, v, o, dout, dq, dk and dv must be 16-byte aligned, rope 8-byte,
 * lse and nvalid 4-byte; other pointers are rejected with ACT_ERR_INVALID before any work is
 * queued. */
#define ACT_NOALLOC_ATTN_SCRATCH_FLOATS (8L * 1024 * 1024)
int act_attention_bwd_noalloc(const void* q, const void* k, const void* v, const void* o, const float* lse,
                              const void* dout, void* dq, void* dk, void* dv, int clips, int T, int Tk, int H,
                              const int32_t* nvalid, int causal, int zero_key, const float* rope, void* stream);
/* Kernel family each launch of the steps issued so far went to, counted as the launches are
 * issued (a captured graph counts once, when it is captured).  counts[i] for i < n receives the
 * count of ACT_PATH_i. */
#define ACT_PATH_ATTN_FWD_TC 0   /* tcgen05 self-attention forward (attention_tc.cu) */
#define ACT_PATH_ATTN_FWD_MMA 1  /* mma.sync attention forward (attention.cu) */
#define ACT_PATH_ATTN_BWD_TC 2   /* tcgen05 self-attention backward */
#define ACT_PATH_ATTN_BWD_MMA 3  /* mma.sync attention backward */
#define ACT_PATH_GEMM_TC 4       /* tcgen05 projection GEMM (gemm_tc.cu) */
#define ACT_PATH_GEMM_MMA 5      /* mma.sync GEMM (gemm_mma.cu) */
#define ACT_PATH_RANK_TC 6       /* tcgen05 rank-block product (gemm_skinny.cu) */
#define ACT_PATH_RANK_MMA 7      /* rank-block product on the mma.sync GEMM */
#define ACT_PATH_XATTN_FWD_TC 8  /* tcgen05 cross-attention forward, <= 64 keys (xattn_tc.cu) */
#define ACT_PATH_XATTN_BWD_TC 9  /* tcgen05 cross-attention backward, <= 64 keys */
#define ACT_PATH_COUNT 10
int act_path_counts(act_ctx* ctx, int64_t* counts, int n);
/* Failure-path check of the device error word (no reference counterpart): one kernel runs the
 * tcgen05 kernels' bounded flag wait on a flag that nothing sets, gives up after limit_ns
 * (1 ns .. 10 s), records its code, and the call returns ACT_ERR_CUDA as a step would after a
 * timed-out wait.  The word is cleared when reported: the context stays usable. */
int act_wait_probe(act_ctx* ctx, int64_t limit_ns);
/* MusicGen: read back the staged delayed inputs ([n][n_q][frames + n_q - 1], build_pattern_sequence
 * of src/mg/pattern.h:64-76 without its last step) and the scored targets ([n][n_q][frames -
 * prefix_frames], src/mg/train.h:195-205) of the last act_mg_stage / act_mg_step. */
int act_mg_staged(act_ctx* ctx, int32_t* ids, size_t n_ids, int32_t* targets, size_t n_targets);
/* MelodyFlow: read back the clean / noise windows of the last act_mf_stage / act_mf_step as the
 * device holds them ([n][latent_dim][frames] each; after on-device sampling, the drawn values). */
int act_mf_staged(act_ctx* ctx, float* clean, float* noise, size_t n_values);
/* Q8_0 blocks (34 bytes: fp16 d, int8 q[32]; tools/ac-quantize.cpp:161) dequantised on the
 * device by the kernels act_bind_weight uses: out_f32 = d * q in fp32, out_f16 = that value
 * rounded to nearest-even f16 (the GEMM operand).  Either output may be NULL. */
int act_q8_0_dequant(int device, const void* blocks, int64_t nblocks, float* out_f32, uint16_t* out_f16);
/* kernels in the captured step graph for microbatch size n (-1 before the graph exists) */
int64_t act_graph_kernel_nodes(act_ctx* ctx, int n);

/* ---- adapter consumption (inference) ---- */
/* lora_linear (src/ac/lora.h:50-83) on host buffers: y [rows][out] (fp32) = W x with the adapter
 * applied as load_lora (src/ac/lora.h:113-170) configures it.  x [rows][in] fp32; W [out][in] of
 * ggml type ACT_TYPE_F32 / F16 / Q8_0 (w_bytes its size); A [rank][in], B [out][rank] fp32, or A
 * NULL for the bare projection; magnitude [out] (DoRA rows) or NULL (LoRA).
 *   LoRA: y = W x + (strength * alpha / rank) B A x
 *   DoRA: y' = (W x + s B A x) * m / sqrt(||W_o||^2 + in*1e-12 + 2s<W_o,(BA)_o> + s^2||(BA)_o||^2),
 *         s = alpha / rank; y = W x + strength (y' - W x)
 * W x runs on the tensor cores (f16 operands: x and F32 weights rounded to f16, Q8_0 dequantised
 * inside the GEMM for more than 128 rows), the rank-sized products in fp32.  in and out must be
 * multiples of 8 (32 for Q8_0), rank <= 64.  Failures: ACT_ERR_INVALID / ACT_ERR_CUDA, message
 * from act_last_error(NULL). */
int act_lora_linear(int device, const float* x, int64_t rows, int in, int out, int w_type, const void* w,
                    size_t w_bytes, const float* A, const float* B, int rank, float alpha, const float* magnitude,
                    float strength, float* y);

/* ---- layer norm with weight gradients, 8-bit activation checkpoints, 8-bit GEMM ----
 * Operators for training more than the adapters keep today: norms whose weight and bias learn,
 * activations kept in 8 bits between forward and backward, and projections whose two operands
 * are 8-bit floating point.  No counterpart in the reference (its norms are frozen, its
 * activations fp32, src/mf/dit.h and src/ac/lora.h).
 *
 * Every pointer is a DEVICE pointer of the calling thread's current device (checked: a host
 * pointer or another device's is rejected), work is queued asynchronously on `stream` (NULL =
 * the legacy default stream), nothing is allocated, and every call may be captured into a CUDA
 * graph.  Tensors are row-major with a row stride in elements (ld >= columns); element types are
 * ACT_TYPE_F32, ACT_TYPE_F16 and ACT_TYPE_BF16, and base pointers are aligned to the element.
 * Any stride and alignment is taken; vectors move when bases, strides and columns are multiples
 * of four elements.  Outputs must not overlap inputs unless said otherwise.  rows = 0 does nothing (and
 * zeroes sums over the rows that are not accumulated); tensors with that many rows, codes and scales
 * among them, may then be NULL, as the address of an empty tensor often is.  The same call gives the same
 * bits every time on the same GPU model: no reduction depends on the order in which blocks finish.
 *
 * An 8-bit tensor is codes and scales.  A block is 128 neighbouring columns (the last one of a
 * row may be shorter) of one row, or of 128 rows for a weight, and has one fp32 scale: the
 * smallest power of two s >= 2^-126 with |x| <= top * s for every finite x of the block (top 448
 * for E4M3, 127 for I8; an all-zero block has 2^-126).  A code is x / s rounded to nearest even,
 * which is exact arithmetic: codes and scales depend on x alone.  Finite values beyond 240 * 2^120 (E4M3) or
 * 127 * 2^121 (I8), the largest that stay finite in fp32, count as those.  Relative to a free scale the
 * power of two costs E4M3 nothing but subnormal range, and I8 at most one bit.  A value that is
 * not finite is stored as NaN (E4M3 code 0x7f, I8 code -128) and leaves its block's scale alone.
 * Scales lie block-major, scale[(column / 128) * lds + row] (row / 128 for blocks of 128 rows):
 * the order in which both products read them. */
#define ACT_CKPT_I8 1   /* whole numbers -127 .. 127: the smaller error, for checkpoints */
#define ACT_CKPT_E4M3 2 /* 8-bit floating point: checkpoints, and operands of act_gemm_f8 */
typedef struct {
    int type;      /* ACT_CKPT_* */
    void* q;       /* codes, one byte each, rows of ldq bytes */
    int64_t ldq;
    float* scale;  /* [ceil(columns / 128)][lds] */
    int64_t lds;
} act_ckpt8;

/* x [rows][cols] -> codes and scales; block_rows 1 (activations) or 128 (weights) */
int act_ckpt8_store(const void* x, int x_type, int64_t ldx, int64_t rows, int64_t cols, int block_rows,
                    const act_ckpt8* out, void* stream);
/* y [rows][cols] = the values codes and scales stand for, rounded to y_type */
int act_ckpt8_load(const act_ckpt8* in, int64_t rows, int64_t cols, int block_rows, void* y, int y_type,
                   int64_t ldy, void* stream);

/* Layer norm of each row: mean, rstd = 1 / sqrt(variance + eps), y = (x - mean) * rstd * w + b in
 * fp32, rounded once to y_type.  w and b are fp32 [dim], each may be NULL (1 and 0).  y may be
 * NULL if y8 is given: y8 (E4M3 or I8, NULL to skip) receives the fp32 result in 8 bits, the
 * operand of act_gemm_f8.  x8 (NULL to skip) receives x itself in 8 bits: the checkpoint
 * act_layernorm_bwd reads in place of x.  mean and rstd are fp32 [rows].  dim <= 8192. */
int act_layernorm_fwd(const void* x, int x_type, int64_t ldx, int64_t rows, int64_t dim, const float* w,
                      const float* b, float eps, void* y, int y_type, int64_t ldy, const act_ckpt8* y8, float* mean,
                      float* rstd, const act_ckpt8* x8, void* stream);
/* Its backward pass, with h = (x - mean) * rstd and dh = dy * w:
 *   dx = rstd * (dh - mean(dh) - h * mean(dh * h)) (+ add),   dw = sum over rows of dy * h,   db = sum of dy.
 * x is given as it was (x_type, ldx) or, with x NULL, as the checkpoint x8.  add (NULL, or
 * dx_type with row stride lddx; dx itself is allowed) is the gradient that reaches x past the
 * norm.  dw and db are fp32 [dim], each may be NULL; accumulate 1 adds to what they hold.
 * workspace: act_layernorm_bwd_workspace bytes, 16-byte aligned, free for reuse once the call's
 * work is done: calls (and captured graphs) that overlap on the GPU need one each. */
int act_layernorm_bwd(const void* dy, int dy_type, int64_t lddy, const void* x, int x_type, int64_t ldx,
                      const act_ckpt8* x8, const float* w, const float* mean, const float* rstd, int64_t rows,
                      int64_t dim, const void* add, void* dx, int dx_type, int64_t lddx, float* dw, float* db,
                      int accumulate, void* workspace, size_t workspace_bytes, void* stream);
/* bytes of workspace for that shape on the current device; -1 for a shape that is refused */
int64_t act_layernorm_bwd_workspace(int64_t rows, int64_t dim);

/* GELU with the checkpoint of its input: g = z * Phi(z) (Phi the normal distribution function),
 * z8 receives z in 8 bits.  g may be NULL if g8 is given (fp32 result in 8 bits, as in
 * act_layernorm_fwd).  g has z's type.  Here and in the backward pass the normal tail is 0 where it would be
 * below 2^-126 (z < -13.2). */
int act_gelu_ckpt8_fwd(const void* z, int z_type, int64_t ldz, int64_t rows, int64_t cols, void* g, int64_t ldg,
                       const act_ckpt8* g8, const act_ckpt8* z8, void* stream);
/* dz = dg * (Phi(z) + z * phi(z)) at the kept z; dz of dg's type may be NULL if dz8 is given. dz may
 * be dg itself. */
int act_gelu_ckpt8_bwd(const void* dg, int dg_type, int64_t lddg, const act_ckpt8* z8, int64_t rows, int64_t cols,
                       void* dz, int64_t lddz, const act_ckpt8* dz8, void* stream);

/* Rank product with a checkpoint, the lora_A gradient (src/ac/lora.h:34-95) from a kept input:
 *   C[j][c] (+)= alpha * sum over rows t of U[t][j] * X[t][c],   C fp32 [nb][cols], 1 <= nb <= 64.
 * X in blocks of 1 row, its scales powers of two as act_ckpt8_store leaves them; its codes start on
 * 16-byte boundaries (q and ldq multiples of 16).  All of U's precision enters the product (fp32 U
 * included) and sums are fp32 (of U and X, what lies below 2^-133, bf16's smallest step, does not count);
 * infinities and NaN in U or X reach C as the formula has them.  accumulate 0 overwrites C.  status: a
 * device int that the caller zeroes once and may read at any time; nonzero means that a bounded wait
 * inside the kernel ran out and C is not valid. */
int act_rank_gemm_ckpt8(const void* u, int u_type, int64_t ldu, int nb, const act_ckpt8* x, int64_t rows,
                        int64_t cols, float alpha, float* c, int64_t ldc, int accumulate, int32_t* status,
                        void* stream);
/* Product of two E4M3 tensors, X [M][K] in blocks of one row and W in blocks of 128 rows:
 *   Y[m][n] = sum over k of X[m][k] * W[n][k] (+ bias[n]) (+ Y[m][n] with accumulate 1).
 * W is stored [N][K] (w_mn_major 0: a projection) or [K][N] (1: the input gradient dY W of a
 * weight [K = out][N = in], the same codes as the projection's).  Scales may be any fp32 values; a
 * block's two are multiplied with each other first.
 * Codes start on 16-byte boundaries (q and ldq multiples of 16).  bias fp32 [N] or NULL.  Sums are
 * fp32.  status as in act_rank_gemm_ckpt8. */
int act_gemm_f8(const act_ckpt8* x, const act_ckpt8* w, int64_t M, int64_t N, int64_t K, int w_mn_major,
                const float* bias, void* y, int y_type, int64_t ldy, int accumulate, int32_t* status, void* stream);

/* Failure-path check of both products' status word: one kernel copies ACT_COPY_PROBE_BYTES from src to
 * dst through shared memory; between the two it waits, as the products do, for something that never
 * comes, gives up after limit_ns (1 ns .. 10 s), writes ACT_COPY_PROBE_CODE to *status (if that is 0)
 * and waits for its copies in flight as they do.  src 16-byte aligned; all three are device pointers. */
#define ACT_COPY_PROBE_BYTES 8192
#define ACT_COPY_PROBE_CODE 98
int act_copy_wait_probe(const void* src, void* dst, int64_t limit_ns, int32_t* status, void* stream);

#if defined(__GNUC__)
#pragma GCC visibility pop
#endif
#ifdef __cplusplus
}
#endif

#endif /* ACTRAIN_H */
