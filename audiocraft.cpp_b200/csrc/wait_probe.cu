// wait_probe.cu -- kernels whose only job is to let a bounded device wait run out.
//
// Every wait in the tcgen05 kernels (mbarrier phases, the stream-K hand-off flag) gives up after
// a time limit, records a code in the context's device error word and returns, so that a wait
// which can never finish ends the kernel instead of hanging the GPU; the host reads the word
// after each step.  This kernel runs the same bounded flag wait on a flag that nothing sets, with
// a caller-chosen limit, so that tests can watch that path end in an error status on a live
// context without faulting or hanging anything.
#include "kernels.h"
#include "tc_common.cuh"

namespace act {

namespace {

__global__ void wait_probe_kernel(const int* flag, unsigned long long limit_ns, int* err) {
    if (threadIdx.x == 0 && blockIdx.x == 0) tc::flag_wait(flag, 1, err, WAIT_PROBE_CODE, limit_ns);
}

// The same for the waits of the kernels whose warps hand registers to each other (gemm_f8.cu,
// rank_ckpt8.cu): a ring of copies is filled, the wait for a barrier that nobody arrives on gives
// up, and the copies are drained as those kernels drain theirs before the CTA may end.
constexpr int PROBE_SLOTS = 2, PROBE_SLOT = COPY_PROBE_BYTES / PROBE_SLOTS;
__global__ void copy_wait_probe_kernel(const char* src, char* dst, unsigned long long limit_ns, int* status) {
    __shared__ __align__(128) char ring[COPY_PROBE_BYTES];
    __shared__ __align__(8) uint64_t bars[PROBE_SLOTS + 1];
    const uint32_t full = smem_u32(bars), never = full + 8 * PROBE_SLOTS;
    if (threadIdx.x == 0) {
        for (int s = 0; s <= PROBE_SLOTS; ++s) tc::mbar_init(full + 8 * s, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        long issued = 0;
        for (int s = 0; s < PROBE_SLOTS; ++s, ++issued) {
            tc::mbar_expect_tx(full + 8 * s, PROBE_SLOT);
            tc::bulk_load(smem_u32(ring) + s * PROBE_SLOT, src + s * PROBE_SLOT, PROBE_SLOT, full + 8 * s);
        }
        tc::mbar_wait_inline(never, 0, status, COPY_PROBE_CODE, limit_ns);
        tc::drain_ring(full, PROBE_SLOTS, issued);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < COPY_PROBE_BYTES; i += blockDim.x) dst[i] = ring[i];
}

}  // namespace

void copy_wait_probe(const void* src, void* dst, long long limit_ns, int* status, cudaStream_t s) {
    copy_wait_probe_kernel<<<1, 128, 0, s>>>(static_cast<const char*>(src), static_cast<char*>(dst),
                                             (unsigned long long)limit_ns, status);
}

void wait_probe(const int* flag, long long limit_ns, int* err, cudaStream_t s) {
    wait_probe_kernel<<<1, 32, 0, s>>>(flag, (unsigned long long)(limit_ns > 0 ? limit_ns : 1), err);
}

}  // namespace act
